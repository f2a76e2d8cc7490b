// Absorbed latent attention on tcgen05: one latent row a token is the key of every head and, without its rotary part, the
// value, so a cached row is read once for all of a sequence's query rows.
//
// A tile of 64 cached rows (TMA, 64-column panels with 128-byte swizzle) meets up to 64 query rows, transposed:
//     S^T = C Q^T        (M = 64 keys, N = query rows, K = R + Dr; both operands K-major)
//     O^T += C^T P^T     (M = 128 latent dims a product, N = query rows, K = 64 keys; both operands MN-major)
// The query rows are the N side because a decode step has few (heads x tokens, padded to 16) and N can be small, and because
// O of 64 rows x 512 dims then takes 4 x 64 of TMEM's 512 columns (as M side it would take all of them for
// 128 rows, and leave none for S). The same tile in shared memory is the A operand of both products. P^T goes
// through 8 KB of shared memory, rows = keys.
//
// Warps: 0 TMA producer, 1 issues the first products (and owns TMEM), 2 the second ones, 3 writes what the join kernel has to know,
// 4-11 softmax and output. S^T uses 16 lanes of each TMEM quadrant; a softmax warp reads its quadrant's 16 keys in the
// 16x256b shape (a thread has two keys of up to four column pairs), warps 4-7 the first half of the columns, 8-11 the second.
// The offset of a query row is raised only when a score exceeds it by more than 2^8, so most tiles need no maximum:
// one vote over the block (a barrier with a reduction) finds that no row grew. Sums stay with each thread until a segment's end.
// What a tile seldom does (raising offsets) and what a segment does once (the output) are loops that are not unrolled: in the way of the
// others, unrolled, their instructions cost fetches and registers (64 sequences of 1k to 32k 207 us with them unrolled, 202 without;
// drafts 40.5 / 35.0; chunks 1105 / 1079).
// Two warps issue so that neither kind of product waits behind one of the other kind that cannot start yet. A tile's panels are loaded
// and freed in two groups, as the second product goes through them.
//
// Work: an item is a block of query rows (tokens x heads of one sequence) over the rows it attends. All items' tiles
// in a row are cut into equal shares, one a CTA, so ragged lengths balance and a long sequence is split where there are
// few; an item that more than one CTA worked on is joined by a second kernel from f32 partial results. Behind a shared
// prefix, rows of several sequences make up an item of their own over the prefix (where a sequence alone fills
// an item, the prefix's tiles simply come first in its own), and every row is joined.
//
// What bounds it: with one token a sequence HBM (64 sequences of 1k to 32k rows of 512 + 64, 16 heads: 202 us, 6.2 TB/s); with 64
// query rows an item the shared memory that feeds the products (a tile of 512 + 64: scores 36 x 33 cycles, outputs 16 x 50,
// its load's writes 576; 509 tokens of 32 heads over 4k to 8k, 4 sequences: 1.08 ms, 770 TFLOP/s, 3050 cycles a tile); with
// smaller rows the chain from scores to weights.
//
// Rows past a sequence's end are zeroed in shared memory before the second product (a weight of 0 would make NaN of
// them). Every mbarrier wait is bounded; the softmax warps, which also meet at block barriers, go on without
// waiting after a timeout so that none is left behind.

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gtb_common.cuh"
#include "latent.h"
#include "latent_mma.cuh"
#include "sdpa_args.h"
#include "sm100_ptx.cuh"

namespace gtb {
namespace {

using namespace sm100;

constexpr int KT = 64;                 // cached rows a tile
constexpr int NR = 64;                 // query rows an item, at most
constexpr int PANEL = KT * 128;        // bytes of 64 rows x 64 columns
constexpr int NTHREADS = 384;
constexpr int NSOFT = 256;             // threads of the softmax warps
constexpr int MAX_STAGES = 6;
constexpr int GROUP = 4;               // panels of a tile's first group; the others (if there are more than 5) are a second one
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t O_COL = 2 * NR;     // S^T buffers at 0 and 64, O^T of dims 128 t .. at O_COL + 64 t
constexpr int SMEM_MAX = 232448;

struct Bars {
    uint64_t q_full, q_empty, pv_done, o_empty, p_full, drain[2], s_free[2];
    uint64_t k_full[2][MAX_STAGES], k_empty[2][MAX_STAGES], s_full[2];
    uint32_t tmem;
    int abort;
};

struct Extra {                 // what lies behind the operands in shared memory
    float alpha[NR];           // factor of a row's sums; at the end 1 / sum
    int out_row[NR];           // row of the output, -1: none
    int lim[NR];               // last own row a query row attends; DEAD: it attends nothing
    float exch[4][NR];         // a quadrant's maxima, later its sums
    Bars bars;
    int64_t line, warp_sum[NTHREADS / 32];  // finding the CTA's share
    int first_item;
    int64_t first_place;
};

constexpr int DEAD = INT_MIN;

struct Params {
    const int32_t *lens, *counts, *prefix_lens;  // counts, prefix_lens nullable
    int64_t Smax, prefix_max;
    int B, H, Lq, R, Dr;
    int hh, ii, n_h, n_rt;     // heads and tokens of an item, items along the heads, items a sequence
    int bb, n_pre;             // sequences of a prefix item (0: the prefix's tiles belong to the own items), prefix items
    int panels, n_groups;
    int q_pitch, q_zero;       // bytes of a panel of Q; whether loads leave some of its rows
    int group_bytes[2], stages[2], slack;
    float scale_log2;
    void* o;
    float* lse;
    float* part_o;             // [slot][row / 4][dim][row % 4]
    float2* part_ml;           // [slot][row]: offset, sum
    int4* joins;               // of each item, or where there are more of them than CTAs, of the item a CTA begins last: item (-1: one
                               // CTA did it all), first CTA, last CTA, tokens of its sequence that attend
    int by_item;
    int* n_used;               // CTAs that have a share
    int lead;                  // places of an item before its tiles'
    int own_rows, own_pitch;   // rows of an own item; the same to a multiple of 16: those of a slot of it
    int join_dims, join_groups;  // warps of a join block along the dims and along the parts
    int64_t own_base;          // first float of own slots in part_o (split prefix)
    int* status;
};

static_assert(3 * 9 * PANEL + PANEL + (int)sizeof(Extra) <= SMEM_MAX, "two stages of the largest rows");

// What an item costs besides its tiles (its query rows' load, the first tile's way through the empty pipeline, its output), in tiles; a
// tile of at most 256 values is about half of one of 512. (32 sequences of 100 to 8192 rows of 256, drafts of 5 tokens of 20 heads: 45.4
// us with 0 places, 40.6 with 2, 34.9 with 3, 34.3 with 5, 34.7 with 8; 12 of 3 to 640 behind 4001, 22.5, 21.0, 20.2, 18.7, 19.1; rows
// of 512, 64 sequences behind 16k: 78.3, 75.3, 76.8, with 4 78.0; chunks of 509 tokens 1101, 1088, 1083, 1083; one token of 64
// sequences of 1k to 32k 203, 202, 202, 204.6.) Between 3 and 5 little changes, and no size between 256 and 512 was measured: the
// border could lie anywhere there.
constexpr int lead_of(int R) { return R <= 256 ? 5 : 3; }

struct Item {
    int b, i0, h0;             // first sequence, token, head
    int nb, ni, nh;            // extent in them (box sizes)
    int len, cnt;              // of an own item's sequence
    int nt_pre, nt;            // tiles over the prefix; tiles in all (at least 1)
    bool pre, empty;           // an item over the prefix alone; no rows to attend
    __device__ __forceinline__ int rows() const { return nb * ni * nh; }
};

__device__ __forceinline__ int prefix_rows(const Params& p) {
    return p.prefix_lens ? (int)min((int64_t)max(p.prefix_lens[0], 0), p.prefix_max) : 0;
}

// items over the prefix alone: only where there are rows in it
__device__ __forceinline__ int prefix_items(const Params& p, int P) { return p.bb && P > 0 ? p.n_pre : 0; }

// where item k lies among the query rows
__device__ __forceinline__ Item item_at(const Params& p, int k, int np) {
    Item it;
    it.nh = p.hh;
    it.ni = p.ii;
    it.pre = k < np;
    if (it.pre) {
        it.b = k * p.bb;
        it.i0 = it.h0 = 0;
        it.nb = p.bb;
    } else {
        k -= np;
        it.nb = 1;
        it.b = k / p.n_rt;
        const int rt = k - it.b * p.n_rt, ti = rt / p.n_h;
        it.i0 = ti * p.ii;
        it.h0 = (rt - ti * p.n_h) * p.hh;
    }
    return it;
}

// and what it attends
__device__ __forceinline__ Item item_of(const Params& p, int k, int P, int np) {
    Item it = item_at(p, k, np);
    const int pt = (P + KT - 1) / KT;
    if (it.pre) {
        it.empty = false;
        it.len = it.cnt = 0;
        it.nt_pre = it.nt = pt;
        return it;
    }
    it.len = (int)min((int64_t)max(p.lens[it.b], 0), p.Smax);
    it.cnt = p.counts ? min(max(p.counts[it.b], 0), p.Lq) : p.Lq;
    const bool live = it.i0 < it.cnt;
    const int keys = live ? max(0, it.len - it.cnt + min(it.i0 + p.ii, it.cnt)) : 0;
    it.nt_pre = live && !p.bb ? pt : 0;
    it.nt = it.nt_pre + (keys + KT - 1) / KT;
    it.empty = it.nt == 0;
    it.nt = max(it.nt, 1);
    return it;
}

// The line: each item takes `lead` places and one for each of its tiles; CTA c of n works on the tiles whose places are in
// [share(c), share(c + 1)).
__device__ __forceinline__ int64_t share(int64_t line, int n, int c) { return line * c / n; }

// the CTA whose share holds place x
__device__ __forceinline__ int cta_of(int64_t line, int n, int64_t x) {
    int c = (int)min((int64_t)n - 1, x * n / line);
    while (c + 1 < n && share(line, n, c + 1) <= x) ++c;
    while (share(line, n, c) > x) --c;
    return c;
}

// query row `col` of an item: (sequence, token, head), false where there is none
__device__ __forceinline__ bool row_of(const Params& p, const Item& it, int col, int& b, int& i, int& h) {
    const int r = col / it.nh;
    h = it.h0 + col - r * it.nh;
    const int s = r / it.ni;
    i = it.i0 + r - s * it.ni;
    b = it.b + s;
    return s < it.nb && h < p.H && i < p.Lq && b < p.B;
}

// slot of CTA c's partial result of item k, in floats of part_o and rows of part_ml
__device__ __forceinline__ void slot_of(const Params& p, int k, int np, int c, bool head, int64_t& o, int64_t& ml) {
    if (!p.bb) {  // a CTA leaves at most two: of the item it begins within, and of the one that it ends within
        const int64_t s = 2 * c + (head ? 1 : 0);
        o = s * p.own_pitch * p.R;
        ml = s * NR;
    } else {      // (a step along the line changes the item or the CTA: k + c names the segment)
        o = k < np ? (int64_t)(k + c) * NR * p.R : p.own_base + (int64_t)(k - np + c) * p.own_pitch * p.R;
        ml = (int64_t)(k + c) * NR;
    }
}

// 16 lanes x 8 n columns of 32 bits (n 1 to 4): of each 8 columns, thread t gets (lane t/4, columns 2 (t%4), +1) and (lane t/4 + 8, the
// same columns)
__device__ __forceinline__ void tmem_ld_16(int n, uint32_t taddr, uint32_t* r) {
    if (n == 1)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(taddr));
    else if (n == 2)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(taddr));
    else  // (of 3 too: the columns behind are allocated, and dropped)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                       "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                     : "r"(taddr));
}

__device__ __forceinline__ void soft_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(NSOFT) : "memory"); }
__device__ __forceinline__ bool soft_any(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "n"(NSOFT)
        : "memory");
    return r != 0;
}

template <bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1)
latent_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQp,
                   const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmCp,
                   const __grid_constant__ Params p) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    if (smem - smem_raw > p.slack) {  // (the largest rows leave less than the alignment may take; it takes nothing)
        if (threadIdx.x == 0) atomicCAS(p.status, 0, 70);
        // the second kernel goes by this table: nothing to join
        const int n = p.by_item ? prefix_items(p, prefix_rows(p)) + p.B * p.n_rt : (int)gridDim.x;
        for (int k = (int)(blockIdx.x * NTHREADS + threadIdx.x); k < n; k += (int)gridDim.x * NTHREADS) p.joins[k] = make_int4(-1, 0, 0, 0);
        if (blockIdx.x == 0 && threadIdx.x == 0) *p.n_used = 0;
        return;
    }
    unsigned char* sQ = smem;
    unsigned char* sC = smem + p.panels * p.q_pitch;  // the stages of the first group, then of the second
    unsigned char* sC1 = sC + p.stages[0] * p.group_bytes[0];
    unsigned char* sP = sC1 + p.stages[1] * p.group_bytes[1];
    Extra& ex = *(Extra*)(sP + PANEL);
    Bars& bar = ex.bars;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
    const int P = prefix_rows(p), np = prefix_items(p, P);
    const int n_items = np + p.B * p.n_rt;

    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full, 1);
        mbar_init(&bar.q_empty, 1);
        mbar_init(&bar.pv_done, 1);
        mbar_init(&bar.o_empty, NSOFT / 32);
        mbar_init(&bar.p_full, NSOFT / 32);
        for (int s = 0; s < 2 * MAX_STAGES; ++s) {
            mbar_init(&bar.k_full[0][0] + s, 1);
            mbar_init(&bar.k_empty[0][0] + s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bar.s_full[s], 1);
            mbar_init(&bar.s_free[s], NSOFT / 32);
            mbar_init(&bar.drain[s], 1);
        }
        bar.abort = 0;
        fence_mbar_init();
    }
    // query rows that no load fills stay zero (their columns are computed and dropped)
    for (int e = threadIdx.x; e < (p.q_zero ? p.panels * p.q_pitch / 16 : 0); e += NTHREADS) ((uint4*)sQ)[e] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    if (warp == 1) tmem_alloc(&bar.tmem, TMEM_COLS);
    // ---------------------------------------------------------------- this CTA's share of the line
    // (NTHREADS items a round; where that is all of them, they are counted once)
    int64_t line = 0, begin = 0, end = 0, before = 0;
    int n_cta = 1;
    for (int pass = n_items > NTHREADS ? 0 : 1; pass < 2; ++pass) {
        for (int k0 = 0; k0 < n_items; k0 += NTHREADS) {
            const int k = k0 + (int)threadIdx.x;
            const int64_t n = k < n_items ? item_of(p, k, P, np).nt + p.lead : 0;
            int64_t incl = n;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(~0u, incl, o);
                if (lane >= o) incl += y;
            }
            if (lane == 31) ex.warp_sum[warp] = incl;
            __syncthreads();
            int64_t total = 0;
            for (int w = 0; w < NTHREADS / 32; ++w) {
                if (w < warp) incl += ex.warp_sum[w];
                total += ex.warp_sum[w];
            }
            incl += before;
            before += total;
            if (pass == 1) {
                if (n_items <= NTHREADS) line = before;
                if (k0 == 0) {
                    n_cta = (int)min((int64_t)gridDim.x, line);
                    if (cta == 0 && threadIdx.x == 0) *p.n_used = n_cta;
                    begin = share(line, n_cta, min(cta, n_cta - 1));
                    end = share(line, n_cta, min(cta, n_cta - 1) + 1);
                }
                if (begin >= incl - n && begin < incl) {
                    ex.first_item = k;
                    ex.first_place = incl - n;
                }
            }
            __syncthreads();
            if (pass == 1 && begin < before) break;  // (begin < line: found by the last round)
        }
        if (pass == 0) line = before, before = 0;
    }
    // from here on places count from the first item's first tile: tiles [off_first, ..) of item k_first, and on to place `last`
    const int k_first = ex.first_item;
    const int64_t first_place = ex.first_place;
    const int off_first = max((int)(begin - first_place) - p.lead, 0), last = (int)(end - first_place) - p.lead;
    const bool idle = cta >= n_cta;

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    volatile int* abort_flag = &bar.abort;
    asm volatile("griddepcontrol.launch_dependents;");  // the join's blocks may take the SMs that this grid's leave
    // A role's walk over the CTA's tiles: for_segments(f) calls f(item, its number, first tile, tiles)
    auto for_segments = [&](auto uni, auto&& f) {
        int to = uni(last), off = uni(off_first);
        for (int k = uni(k_first); k < n_items && !idle; ++k, off = 0) {
            const Item it = item_of(p, k, P, np);
            const int n = uni(min(it.nt, to) - off);
            if (n <= 0) break;
            to -= uni(it.nt) + p.lead;
            if (!f(it, k, off, n)) break;
        }
    };
    auto plain = [](int v) { return v; };

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            prefetch_tmap(&tmQ);
            prefetch_tmap(&tmC);
            bool ok = true;
            int nseg = 0, loads[2] = {0, 0};  // segments started, groups loaded
            int stage[2] = {0, 0}, phase[2] = {1, 1};
            for_segments(plain, [&](const Item& it, int, int off, int n) {
                if (it.empty) return true;
                for (int t = off; t < off + n && ok; ++t) {
                    const bool pre = t < it.nt_pre;
                    const CUtensorMap* tm = pre ? &tmCp : &tmC;
                    const int row = (pre ? t : t - it.nt_pre) * KT, b = pre ? 0 : it.b;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        if (!ok || g >= p.n_groups) continue;
                        const int s = stage[g];
                        if (loads[g] >= p.stages[g]) ok = mbar_wait(&bar.k_empty[g][s], phase[g], p.status, 71);
                        if (!ok || *abort_flag) { ok = false; continue; }
                        mbar_expect_tx(&bar.k_full[g][s], p.group_bytes[g]);
                        unsigned char* dst = (g ? sC1 : sC) + s * p.group_bytes[g];
                        for (int a = 0; a < p.group_bytes[g] / PANEL; ++a)
                            tma_load_4d(dst + a * PANEL, tm, (GROUP * g + a) * 64, row, b, 0, &bar.k_full[g][s]);
                        ++loads[g];
                        if (++stage[g] == p.stages[g]) stage[g] = 0, phase[g] ^= 1;
                    }
                    if (!ok) break;
                    if (t == off) {  // the segment's query rows, once the last one's have been read
                        if (nseg > 0) ok = mbar_wait(&bar.q_empty, (nseg - 1) & 1, p.status, 72);
                        if (!ok || *abort_flag) { ok = false; break; }
                        mbar_expect_tx(&bar.q_full, it.rows() * 128 * p.panels);
                        for (int a = 0; a < p.panels; ++a)
                            tma_load_4d(sQ + a * p.q_pitch, it.pre ? &tmQp : &tmQ, a * 64, it.h0, it.i0, it.b, &bar.q_full);
                        ++nseg;
                    }
                }
                return ok;
            });
            if (!ok) *abort_flag = 1;
            if (*abort_flag) {  // our copies in flight end before the CTA does
                if (nseg > 0) mbar_wait(&bar.q_full, (nseg - 1) & 1, nullptr, 0);
                for (int g = 0; g < p.n_groups; ++g)
                    for (int v = max(0, loads[g] - p.stages[g]); v < loads[g]; ++v)
                        mbar_wait(&bar.k_full[g][v % p.stages[g]], (v / p.stages[g]) & 1, nullptr, 0);
            }
        }
    } else if (warp < 3) {
        // ------------------------------------------------------------ MMA issuers: 1 the scores, 2 the second products
        const bool scores = warp == 1, lead = elect_lane();
        const uint32_t tm = (uint32_t)uniform((int)tmem);
        const uint32_t lead_off = scores ? 16 : PANEL;  // leading byte offset (K-major: unused)
        const uint32_t qd = (uint32_t)desc_sw128(smem_u32(sQ), 16, 1024), pd = (uint32_t)desc_sw128(smem_u32(sP), PANEL, 1024);
        const uint32_t cd[2] = {(uint32_t)desc_sw128(smem_u32(sC), lead_off, 1024), (uint32_t)desc_sw128(smem_u32(sC1), lead_off, 1024)};
        const uint32_t q_step = p.q_pitch >> 4;
        const int rope_steps = p.Dr / 16, m_tiles = (p.R + 127) / 128;
        bool ok = true;
        int nseg = 0;
        int u = 0, stage[2] = {0, 0}, phase[2] = {0, 0};  // tiles so far, the next one's stages and their phases
        for_segments([](int v) { return uniform(v); }, [&](const Item& it, int, int, int n) {
            if (uniform(it.empty)) return true;
            const uint32_t n16 = uniform((it.rows() + 15) & ~15);
            if (scores) {
                const uint32_t idesc = idesc_f16(KT, 0, BF16, false) | (n16 >> 3 << 17);
                ok = warp_wait(&bar.q_full, nseg & 1, p.status, 74);
                for (int t = 0; t < n && ok; ++t, ++u) {
                    if (u >= 2) ok = warp_wait(&bar.s_free[u & 1], ((u >> 1) - 1) & 1, p.status, 75);
                    if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
                    const uint32_t dst = tm + (u & 1) * NR;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        if (!ok || g >= p.n_groups) continue;
                        ok = warp_wait(&bar.k_full[g][stage[g]], phase[g], p.status, 73);
                        if (!ok) continue;
                        tc_fence_after();
                        const uint32_t a = uniform(cd[g] + stage[g] * (p.group_bytes[g] >> 4)), q = qd + GROUP * g * q_step;
                        const int n_val = min(GROUP, p.panels - 1 - GROUP * g);  // panels of latent values
                        if (lead) {
#pragma unroll
                            for (int i = 0; i < GROUP; ++i) {
                                if (i < n_val) {
#pragma unroll
                                    for (int kk = 0; kk < 4; ++kk)
                                        mma_ss_lo(dst, a + i * (PANEL >> 4) + kk * 2, q + i * q_step + kk * 2, idesc, i > 0 || kk > 0 || g > 0);
                                }
                            }
                            if (g + 1 == p.n_groups)  // the rotary keys
                                for (int kk = 0; kk < rope_steps; ++kk)
                                    mma_ss_lo(dst, a + n_val * (PANEL >> 4) + kk * 2, q + n_val * q_step + kk * 2, idesc, 1);
                        }
                        if (++stage[g] == p.stages[g]) stage[g] = 0, phase[g] ^= 1;
                    }
                    if (!ok) break;
                    if (lead) {
                        mma_commit(&bar.s_full[u & 1]);
                        if (t + 1 == n) mma_commit(&bar.q_empty);
                    }
                }
            } else {
                const uint32_t idesc = idesc_f16_amn(128, 0, BF16, true) | (n16 >> 3 << 17);
                // the segment's first product overwrites O^T: the last one's epilogue must have read it
                if (nseg > 0) ok = warp_wait(&bar.o_empty, (nseg - 1) & 1, p.status, 76);
                for (int t = 0; t < n && ok; ++t, ++u) {
                    ok = warp_wait(&bar.p_full, u & 1, p.status, 81);
                    if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t a0 = uniform(cd[0] + stage[0] * (p.group_bytes[0] >> 4));
                    const uint32_t a1 = uniform(cd[1] + stage[1] * (p.group_bytes[1] >> 4));
                    if (lead) {
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            if (m < m_tiles) {
#pragma unroll
                                for (int kk = 0; kk < KT / 16; ++kk)
                                    mma_ss_lo(tm + O_COL + m * NR, (m < 2 ? a0 : a1) + (m & 1) * (2 * PANEL >> 4) + kk * 128, pd + kk * 128, idesc,
                                        t > 0 || kk > 0);
                                if (m == 1 && p.n_groups > 1) mma_commit(&bar.k_empty[0][stage[0]]);
                            }
                        }
                        if (p.n_groups > 1) mma_commit(&bar.k_empty[1][stage[1]]);
                        else mma_commit(&bar.k_empty[0][stage[0]]);
                        mma_commit(&bar.pv_done);
                    }
#pragma unroll
                    for (int g = 0; g < 2; ++g)
                        if (++stage[g] == p.stages[g]) stage[g] = 0;
                }
            }
            ++nseg;
            return ok;
        });
        if (!ok) *abort_flag = 1;
        __syncwarp();
        if (__any_sync(~0u, *abort_flag)) {
            if (lead) mma_commit(&bar.drain[warp - 1]);
            warp_wait(&bar.drain[warp - 1], 0, nullptr, 0);
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------ what the join kernel has to know
        if (lane == 0) {
            int4 mine = make_int4(-1, 0, 0, 0);
            int64_t place = first_place + p.lead;  // of the item's first tile
            for_segments(plain, [&](const Item& it, int k, int off, int) {
                if (off == 0) {
                    const int to = cta_of(line, n_cta, place + it.nt - 1);
                    const bool parts = p.bb ? !it.empty : to > cta;  // (behind a split prefix all rows are joined)
                    const int4 j = make_int4(parts ? k : -1, cta, to, it.cnt);
                    if (p.by_item) p.joins[k] = j;
                    else if (parts) mine = j;
                }
                place += it.nt + p.lead;
                return true;
            });
            if (!p.by_item && !idle) p.joins[cta] = mine;
        }
    } else {
        // ------------------------------------------------------------ softmax, rescaling, epilogue
        const int st = (int)threadIdx.x - 128, quad = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        const int key0 = quad * 16 + (lane >> 2);          // this thread's keys of a tile: key0, key0 + 8
        const int cpair = 2 * (lane & 3);                  // its columns of a group: cpair, cpair + 1
        const int m_tiles = (p.R + 127) / 128;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
        bool ok = true;
        int u = 0, stage[2] = {0, 0};
        for_segments(plain, [&](const Item& it, int k, int off, int n) {
            const int gl = (it.rows() + 15) / 16;          // groups of 8 columns of this warp: 2 j + half, j < gl
            soft_sync();                                   // the last segment's lim, out_row, alpha have been read
            if (st < NR) {
                int b, i, h;
                const bool is = row_of(p, it, st, b, i, h);
                ex.out_row[st] = is ? (b * p.H + h) * p.Lq + i : -1;
                ex.lim[st] = !is || it.pre ? INT_MAX : i >= it.cnt ? DEAD : it.len - it.cnt + i;
            }
            soft_sync();
            const int lim_min = it.len - it.cnt + it.i0;   // smallest limit of a live row
            // a row's state: minus its offset (0 before it has one), what its scores less the offset may reach without a new one, its sum
            float nm[4][2], thr[4][2], l[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int c = 0; c < 2; ++c) nm[j][c] = l[j][c] = 0.0f, thr[j][c] = -INFINITY;
            // one tile, of GL groups of 8 columns a warp
            auto tile = [&](auto groups, int t) {
                constexpr int GL = decltype(groups)::value;
                const bool pre = t < it.nt_pre;
                const int row0 = (pre ? t : t - it.nt_pre) * KT;
                const int valid = (pre ? P : it.len) - row0;  // cached rows of the tile
                if (ok) ok = warp_wait(&bar.s_full[u & 1], (u >> 1) & 1, p.status, 77);
                tc_fence_after();
                uint32_t raw[16];
                float (*e)[4] = (float(*)[4])raw;
                auto scores = [&]() {  // the thread's scores, -inf where the row does not attend the key
                    tmem_ld_16(GL, tmem + lane_addr + (u & 1) * NR + 8 * half * GL, raw);
                    tmem_ld_wait();
                    if (pre ? valid < KT : row0 + KT - 1 > lim_min) {
#pragma unroll
                        for (int j = 0; j < GL; ++j) {
                            const int c = 8 * (half * GL + j) + cpair;
                            // (rows that attend nothing take the others' way and are dropped at the end)
                            const int l0 = pre ? P - 1 : max(ex.lim[c], -1), l1 = pre ? P - 1 : max(ex.lim[c + 1], -1);
                            if (row0 + key0 > l0) e[j][0] = -INFINITY;
                            if (row0 + key0 > l1) e[j][1] = -INFINITY;
                            if (row0 + key0 + 8 > l0) e[j][2] = -INFINITY;
                            if (row0 + key0 + 8 > l1) e[j][3] = -INFINITY;
                        }
                    }
                };
                // (score - offset) * scale: the difference first, so that scores of any size keep what they differ by
                auto exponents = [&]() {
#pragma unroll
                    for (int j = 0; j < GL; ++j)
#pragma unroll
                        for (int c = 0; c < 4; c += 2)
                            f2_unpack(f2_mul(f2_add(f2_pack(e[j][c], e[j][c + 1]), f2_pack(nm[j][0], nm[j][1])), sc2), e[j][c], e[j][c + 1]);
                };
                scores();
                exponents();
                bool grow = false;
#pragma unroll
                for (int j = 0; j < GL; ++j)
#pragma unroll
                    for (int c = 0; c < 2; ++c) grow = grow || fmaxf(e[j][c], e[j][c + 2]) > thr[j][c];
                if (__builtin_expect(soft_any(grow), 0)) {
                    // the rows' maxima over the tile: over the thread's two keys, the warp's 16, the four quadrants
                    scores();
#pragma unroll
                    for (int j = 0; j < GL; ++j) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float v = fmaxf(e[j][c], e[j][c + 2]);
                            v = fmaxf(v, __shfl_xor_sync(~0u, v, 4));
                            v = fmaxf(v, __shfl_xor_sync(~0u, v, 8));
                            v = fmaxf(v, __shfl_xor_sync(~0u, v, 16));
                            if (lane < 4) ex.exch[quad][8 * (half * GL + j) + cpair + c] = v;
                        }
                    }
                    soft_sync();
#pragma unroll
                    for (int j = 0; j < GL; ++j) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int col = 8 * (half * GL + j) + cpair + c;
                            const float v = fmaxf(fmaxf(ex.exch[0][col], ex.exch[1][col]), fmaxf(ex.exch[2][col], ex.exch[3][col]));
                            const float m = thr[j][c] == -INFINITY ? -INFINITY : -nm[j][c], mn = fmaxf(m, v);
                            const float al = mn == m ? 1.0f : ex2((m - mn) * p.scale_log2);
                            if (mn > -INFINITY) nm[j][c] = -mn, thr[j][c] = 8.0f;
                            l[j][c] *= al;
                            if (quad == 0 && lane < 4) ex.alpha[col] = al;
                        }
                    }
                    if (t > off) {  // O^T takes the same factors, once the last tile's product has been added
                        if (ok) ok = warp_wait(&bar.pv_done, (u - 1) & 1, p.status, 78);
                        soft_sync();
                        tc_fence_after();
                        for (int mt = half; mt < m_tiles; mt += 2) {
#pragma unroll 1
                            for (int j = 0; j < GL; ++j) {
                                uint32_t v[16];
                                tmem_ldx<16>(tmem + lane_addr + O_COL + mt * NR + 16 * j, v);
                                tmem_ld_wait();
#pragma unroll
                                for (int c = 0; c < 16; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * ex.alpha[16 * j + c]);
                                tmem_st16(tmem + lane_addr + O_COL + mt * NR + 16 * j, v);
                            }
                        }
                        tmem_st_wait();
                    }
                    exponents();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.s_free[u & 1]);
                uint32_t w[GL][2];
#pragma unroll
                for (int j = 0; j < GL; ++j) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) e[j][c] = ex2(e[j][c]);
                    l[j][0] += e[j][0] + e[j][2];
                    l[j][1] += e[j][1] + e[j][3];
                    w[j][0] = pack2<BF16>(e[j][0], e[j][1]);
                    w[j][1] = pack2<BF16>(e[j][2], e[j][3]);
                }
                if (u > 0 && ok) ok = warp_wait(&bar.pv_done, (u - 1) & 1, p.status, 79);  // P's buffer is free
#pragma unroll
                for (int j = 0; j < GL; ++j) {
                    unsigned char* d = sP + key0 * 128 + (((half * GL + j) ^ (key0 & 7)) << 4) + cpair * 2;
                    *(uint32_t*)d = w[j][0];
                    *(uint32_t*)(d + 8 * 128) = w[j][1];
                }
                if (valid < KT) {  // rows past the end: 0 in the second product, whatever they hold
                    const int first = max(valid, 0), per = (KT - first) * 8;
#pragma unroll 1
                    for (int i = st; i < per * (p.R / 64); i += NSOFT) {
                        const int a = i / per, r = i - a * per, g = a >= GROUP && p.n_groups > 1;
                        unsigned char* base = (g ? sC1 : sC) + stage[g] * p.group_bytes[g];
                        *(uint4*)(base + (a - GROUP * g) * PANEL + first * 128 + r * 16) = make_uint4(0, 0, 0, 0);
                    }
                }
#pragma unroll
                for (int g = 0; g < 2; ++g)
                    if (++stage[g] == p.stages[g]) stage[g] = 0;
                fence_proxy_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.p_full);
            };
            auto tiles = [&](auto groups) {
#pragma unroll 1
                for (int t = off; t < off + n; ++t, ++u) tile(groups, t);
            };
            if (it.empty) {
            } else if (gl == 1) {
                tiles(std::integral_constant<int, 1>{});
            } else if (gl == 2) {
                tiles(std::integral_constant<int, 2>{});
            } else if (gl == 3) {
                tiles(std::integral_constant<int, 3>{});
            } else {
                tiles(std::integral_constant<int, 4>{});
            }
            // ---- the segment's rows: sums over the quadrants, then O^T a latent dim a lane
            // (written over the last tile's maxima and factors: no vote of a next tile lies between, and a warp may still read them)
            soft_sync();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= gl) continue;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float v = l[j][c];
                    v += __shfl_xor_sync(~0u, v, 4);
                    v += __shfl_xor_sync(~0u, v, 8);
                    v += __shfl_xor_sync(~0u, v, 16);
                    if (lane < 4) ex.exch[quad][8 * (half * gl + j) + cpair + c] = v;
                    if (quad == 0 && lane < 4) ex.alpha[8 * (half * gl + j) + cpair + c] = thr[j][c] == -INFINITY ? -INFINITY : -nm[j][c] * p.scale_log2;
                }
            }
            soft_sync();
            const bool whole = !p.bb && off == 0 && n == it.nt;
            int64_t so, sml;
            slot_of(p, k, np, cta, off == 0, so, sml);
            float lsum = 0.0f, mrow = -INFINITY;
            if (st < NR) {
                mrow = ex.alpha[st];
                lsum = (ex.exch[0][st] + ex.exch[1][st]) + (ex.exch[2][st] + ex.exch[3][st]);
                if (ex.lim[st] == DEAD || it.empty || st >= gl * 16) lsum = 0.0f, mrow = -INFINITY;
            }
            soft_sync();
            if (st < NR && ex.out_row[st] >= 0) {
                ex.alpha[st] = lsum == 0.0f ? 0.0f : 1.0f / lsum;  // (NaN stays NaN)
                if (whole) {
                    if (p.lse && ok) p.lse[ex.out_row[st]] = lsum == 0.0f ? -INFINITY : (mrow + log2f(lsum)) * 0.69314718055994531f;
                } else if (ok) {
                    p.part_ml[sml + st] = make_float2(mrow, lsum);
                }
            }
            if (!it.empty && ok) ok = warp_wait(&bar.pv_done, (u - 1) & 1, p.status, 80);
            soft_sync();
            tc_fence_after();
            for (int mt = half; mt < m_tiles; mt += 2) {
                const int d = mt * 128 + quad * 32 + lane;
#pragma unroll 1
                for (int j = 0; j < gl; ++j) {
                    uint32_t v[16];
                    tmem_ldx<16>(tmem + lane_addr + O_COL + mt * NR + 16 * j, v);
                    tmem_ld_wait();
                    if (mt * 128 + quad * 32 >= p.R || !ok) continue;  // (the same for the warp)
                    if (whole) {
                        // 16 rows of one dim a lane become 4 rows of 4 dims: with the neighbour's and then with the
                        // next pair's, each giving away the half of the rows that the other keeps
                        uint32_t w[8];
#pragma unroll
                        for (int c = 0; c < 16; c += 4) {
                            const float4 f = *(const float4*)(ex.alpha + 16 * j + c);  // 0: nothing attended, whatever O^T holds
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float g = e == 0 ? f.x : e == 1 ? f.y : e == 2 ? f.z : f.w;
                                v[c + e] = __float_as_uint(g == 0.0f ? 0.0f : __uint_as_float(v[c + e]) * g);
                            }
                        }
                        const bool odd = lane & 1, far = lane & 2;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const float mine = __uint_as_float(odd ? v[8 + c] : v[c]);
                            const float other = __shfl_xor_sync(~0u, __uint_as_float(odd ? v[c] : v[8 + c]), 1);
                            w[c] = odd ? pack2<BF16>(other, mine) : pack2<BF16>(mine, other);
                        }
                        uint2 y[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t mine = far ? w[4 + c] : w[c], other = __shfl_xor_sync(~0u, far ? w[c] : w[4 + c], 2);
                            y[c] = far ? make_uint2(other, mine) : make_uint2(mine, other);
                        }
                        const int4 r = *(const int4*)(ex.out_row + 16 * j + 8 * odd + 4 * far);
                        T* o = (T*)p.o + (d & ~3);
                        if (r.x >= 0) *(uint2*)(o + (int64_t)r.x * p.R) = y[0];
                        if (r.y >= 0) *(uint2*)(o + (int64_t)r.y * p.R) = y[1];
                        if (r.z >= 0) *(uint2*)(o + (int64_t)r.z * p.R) = y[2];
                        if (r.w >= 0) *(uint2*)(o + (int64_t)r.w * p.R) = y[3];
                    } else if (!it.empty) {
                        uint4* y = (uint4*)(p.part_o + so) + 4 * j * p.R + d;
#pragma unroll
                        for (int c = 0; c < 4; ++c) y[c * p.R] = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (!it.empty && lane == 0) mbar_arrive(&bar.o_empty);
            return true;
        });
        if (!ok) *abort_flag = 1;
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// Rows whose item more than one CTA worked on. A block has 4 rows (a vector of the parts' layout). A warp has 32 E dims, E a lane;
// join_dims warps lie along the dims, join_groups of them take the parts in turn. E = 4 where that gives enough blocks, E = 1 and all
// warps along the parts where a few sequences were cut into many.
// What it costs is latency: of two dependent loads (which parts, then the parts), and of fetching its instructions, which
// each SM runs about once. So what does not depend on the first kernel comes before the wait for it, loops that mostly run once are not
// unrolled, and rows that begin within a vector have a loop of their own (32 sequences of 100 to 8192 rows, drafts of 5 tokens of 20
// heads: issuing the first loads 0.4 instead of 2.7 us, the call 39.8 instead of 44.6).
constexpr int JOIN_WARPS = 8, JOIN_ROWS = 4, JOIN_FLIGHT = 4;
constexpr int MAX_CTAS = 511;  // parts of a row: one a CTA, and one more behind a split prefix

template <typename T, int E>
__global__ void __launch_bounds__(JOIN_WARPS * 32, E == 1 ? 4 : 2) latent_join_kernel(const __grid_constant__ Params p) {
    __shared__ float4 sum[JOIN_WARPS][E][32];
    __shared__ float2 sh_ml[(MAX_CTAS + 1) * JOIN_ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col0 = (int)blockIdx.y * JOIN_ROWS;
    const int np = p.bb ? prefix_items(p, prefix_rows(p)) : 0, rows = min(JOIN_ROWS, p.own_rows - col0);
    const int groups = p.join_groups, group = warp / p.join_dims;
    const int d = ((int)blockIdx.z * p.join_dims + warp % p.join_dims) * 32 * E + lane;  // and every 32nd behind it, E of them
    int orow = -1, token = 0;  // lanes 0 .. 3: the rows' places in the output
    auto place = [&](int k) {
        if (lane >= rows) return;
        int b, h;
        if (row_of(p, item_at(p, k, np), col0 + lane, b, token, h)) orow = (b * p.H + h) * p.Lq + token;
    };
    if (p.by_item) place(np + (int)blockIdx.x);
    const int pre_item = p.bb ? (int)blockIdx.x / p.bb : 0, pre_row = ((int)blockIdx.x - pre_item * p.bb) * p.own_rows + col0;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the first kernel ends
    // parts: CTAs c0 .. c0 + n - 1 of item k, its rows from `row` on; with a split prefix those of the prefix's item come first
    int k[2], c0[2], n[2] = {0, 0}, row[2], cnt;
    if (!p.bb) {
        const int4 j = p.joins[blockIdx.x];
        if (!p.by_item && (int)blockIdx.x >= *p.n_used) return;
        if (j.x < 0) return;
        if (!p.by_item) place(j.x);
        k[0] = j.x, c0[0] = j.y, n[0] = j.z - j.y + 1, row[0] = col0, cnt = j.w;
        k[1] = c0[1] = row[1] = 0;
    } else {
        const int4 own = p.joins[np + (int)blockIdx.x], pre = np > 0 ? p.joins[pre_item] : make_int4(-1, 0, 0, 0);
        k[0] = pre.x, c0[0] = pre.y, n[0] = pre.x < 0 ? 0 : pre.z - pre.y + 1, row[0] = pre_row;
        k[1] = own.x, c0[1] = own.y, n[1] = own.x < 0 ? 0 : own.z - own.y + 1, row[1] = col0;
        cnt = own.w;
    }
    const int parts = n[0] + n[1];
    // where a source's first part is, and the step from CTA to CTA (one address a part: with all of it formed each time, instructions
    // were what this kernel waited for)
    const float* o0[2];
    const float2* ml0[2];
    int o_step[2];
    const int ml_step = (p.bb ? 1 : 2) * NR;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        int64_t so, sml;
        slot_of(p, k[s], np, c0[s], false, so, sml);
        const int pitch = k[s] < np ? NR : p.own_pitch;
        o0[s] = p.part_o + so + ((row[s] >> 2) * p.R + d) * 4;
        ml0[s] = p.part_ml + sml + row[s];
        o_step[s] = (p.bb ? 1 : 2) * pitch * p.R;
    }
    auto load = [&](int q0, float4 (*y)[E]) {  // this lane's dims of parts q0, q0 + groups, ..
#pragma unroll
        for (int e = 0; e < JOIN_FLIGHT; ++e) {
            const int q = q0 + groups * e, s = q >= n[0], i = q - (s ? n[0] : 0), step = s ? o_step[1] : o_step[0];
            // (without a split prefix, the CTA that begins the item has it in its second slot)
            const float* o = (s ? o0[1] : o0[0]) + i * step + (i == 0 && !p.bb ? step / 2 : 0);
            if (q < parts) {
#pragma unroll
                for (int c = 0; c < E; ++c)
                    if (d + 32 * c < p.R) y[e][c] = *(const float4*)(o + 128 * c);
            }
        }
    };
    // a prefix item's rows of a sequence may begin within a vector: `skew` rows into it
    const int skew = row[0] & 3, first = (skew ? n[0] : 0) + group;
    float4 y[JOIN_FLIGHT][E];
    load(first, y);  // (out before the offsets and sums are asked for)
#pragma unroll 1
    for (int e = threadIdx.x; e < parts * JOIN_ROWS; e += blockDim.x) {
        const int q = e / JOIN_ROWS, r = e % JOIN_ROWS, s = q >= n[0], i = q - (s ? n[0] : 0);
        sh_ml[e] = r < rows ? (s ? ml0[1] : ml0[0])[i * ml_step + (i == 0 && !p.bb ? NR : 0) + r] : make_float2(-INFINITY, 0.0f);
    }
    __syncthreads();
    // the rows' largest offset and the sum in its terms: a row a lane & 3, 8 parts at a time
    float m = -INFINITY, l = 0.0f;
#pragma unroll 1
    for (int e = lane; e < parts * JOIN_ROWS; e += 32) m = fmaxf(m, sh_ml[e].x);
    for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, x));
    auto factor = [&](float2 v) { return v.y == 0.0f ? 0.0f : ex2(v.x - m); };  // (a part without a weight holds nothing)
#pragma unroll 1
    for (int e = lane; e < parts * JOIN_ROWS; e += 32) l += sh_ml[e].y * factor(sh_ml[e]);
    for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(~0u, l, x);
    float acc[E][JOIN_ROWS] = {};
    if (skew) {
#pragma unroll 1
        for (int q = group; q < n[0]; q += groups) {
            const float f = factor(sh_ml[q * JOIN_ROWS + (lane & 3)]);
            const float* o = o0[0] + q * o_step[0];
#pragma unroll 1
            for (int r = 0; r < rows; ++r) {
                const float fr = __shfl_sync(~0u, f, r);
                const float* x = o + ((skew + r) >> 2) * p.R * 4 + ((skew + r) & 3);
                if (fr == 0.0f) continue;
#pragma unroll
                for (int c = 0; c < E; ++c) {
                    const float v = d + 32 * c < p.R ? x[128 * c] * fr : 0.0f;
                    acc[c][0] += r == 0 ? v : 0.0f, acc[c][1] += r == 1 ? v : 0.0f, acc[c][2] += r == 2 ? v : 0.0f, acc[c][3] += r == 3 ? v : 0.0f;
                }
            }
        }
    }
#pragma unroll 1
    for (int q0 = first; q0 < parts; q0 += groups * JOIN_FLIGHT) {
        // factor of part q0 + groups * e and row r in lane 4 e + r
        const int q = q0 + groups * (lane >> 2);
        const float f = lane < 4 * JOIN_FLIGHT && q < parts ? factor(sh_ml[q * JOIN_ROWS + (lane & 3)]) : 0.0f;
#pragma unroll
        for (int e = 0; e < JOIN_FLIGHT; ++e) {
#pragma unroll
            for (int r = 0; r < JOIN_ROWS; ++r) {
                const float fr = __shfl_sync(~0u, f, 4 * e + r);
                if (fr != 0.0f) {
#pragma unroll
                    for (int c = 0; c < E; ++c) acc[c][r] = fmaf(r == 0 ? y[e][c].x : r == 1 ? y[e][c].y : r == 2 ? y[e][c].z : y[e][c].w, fr, acc[c][r]);
                }
            }
        }
        load(q0 + groups * JOIN_FLIGHT, y);
    }
    if (groups > 1) {
#pragma unroll
        for (int c = 0; c < E; ++c) sum[warp][c][lane] = make_float4(acc[c][0], acc[c][1], acc[c][2], acc[c][3]);
        __syncthreads();
        if (group > 0) return;
#pragma unroll 1
        for (int g = 1; g < groups; ++g) {
#pragma unroll
            for (int c = 0; c < E; ++c) {
                const float4 z = sum[g * p.join_dims + warp][c][lane];
                acc[c][0] += z.x;
                acc[c][1] += z.y;
                acc[c][2] += z.z;
                acc[c][3] += z.w;
            }
        }
    }
    // what the rows' sums are multiplied by (0: nothing attended)
    float inv = 0.0f;
    if (orow >= 0) {
        const bool none = token >= cnt || l == 0.0f;
        if (!none) inv = 1.0f / l;
        if (p.lse && blockIdx.z == 0 && warp == 0) p.lse[orow] = none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
#pragma unroll
    for (int r = 0; r < JOIN_ROWS; ++r) {
        const int to = __shfl_sync(~0u, orow, r);
        const float f = __shfl_sync(~0u, inv, r);
        T* o = (T*)p.o + (int64_t)to * p.R + d;
#pragma unroll
        for (int c = 0; c < E; ++c)
            if (to >= 0 && d + 32 * c < p.R) Elem<T>::store(o + 32 * c, f == 0.0f ? 0.0f : acc[c][r] * f);
    }
}

// nothing cached and nothing before it: zeros and -inf
__global__ void latent_nothing_kernel(uint16_t* o, int64_t n, float* lse, int64_t rows) {
    const int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = e; i < n; i += step) o[i] = 0;
    for (int64_t i = e; lse && i < rows; i += step) lse[i] = -INFINITY;
}

// 4-D map of 16-bit values with a 64-column box and 128-byte swizzle; sizes and strides (elements) from the second dimension on
bool make_map(CUtensorMap* tm, const void* base, bool bf16, int64_t cols, const int64_t (&size)[3], const int64_t (&stride)[3],
              const int (&box)[3]) {
    if (!encode_fn()) {
        set_error("latent_attention: cuTensorMapEncodeTiled is unavailable");
        return false;
    }
    cuuint64_t dims[4] = {(cuuint64_t)cols, (cuuint64_t)size[0], (cuuint64_t)size[1], (cuuint64_t)size[2]}, st[3];
    for (int i = 0; i < 3; ++i) {
        const int64_t bytes = (size[i] == 1 ? (cols + 7) / 8 * 8 : stride[i]) * 2;  // (a dimension of size 1 is never stepped)
        if (bytes <= 0 || bytes % 16 || bytes >= (1ll << 40)) {
            set_error("latent_attention: a stride is not a positive multiple of 16 bytes below 2^40");
            return false;
        }
        st[i] = (cuuint64_t)bytes;
    }
    const cuuint32_t bx[4] = {64, (cuuint32_t)box[0], (cuuint32_t)box[1], (cuuint32_t)box[2]};
    const CUresult r = encode_tiled_4d(tm, bf16, (void*)base, dims, st, bx);
    if (r != CUDA_SUCCESS) {
        set_errorf("latent_attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
        return false;
    }
    return true;
}

template <bool BF16>
int launch(const LatentAttnArgs& a, cudaStream_t st) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    const char* ctx = "latent_attention";
    int dev = 0, n_sm = 0;
    if (cuda_failed(cudaGetDevice(&dev), ctx) || cuda_failed(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev), ctx))
        return -1;
    Params p{};
    p.lens = a.c.lens;
    p.counts = a.counts;
    p.Smax = a.c.Smax;
    p.B = (int)a.c.B;
    p.H = (int)a.H;
    p.Lq = (int)a.Lq;
    p.R = a.c.R;
    p.Dr = a.c.Dr;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.o = a.o;
    p.lse = a.lse;
    p.status = a.status;
    if (a.prefix.rows) {
        p.prefix_lens = a.prefix.lens;
        p.prefix_max = a.prefix.Smax;
    }
    // rows of an item: all heads of as many tokens as fit, or a part of the heads of one token, in equal parts
    p.n_h = (p.H + NR - 1) / NR;
    p.hh = (p.H + p.n_h - 1) / p.n_h;
    const int fit = p.n_h > 1 ? 1 : NR / p.hh, n_i = (p.Lq + fit - 1) / fit;
    p.ii = (p.Lq + n_i - 1) / n_i;
    p.n_rt = n_i * p.n_h;
    const int own_rows = p.hh * p.ii;
    p.own_rows = own_rows;
    p.own_pitch = (own_rows + 15) & ~15;
    // a prefix gets items of its own where those can take the rows of several sequences
    if (a.prefix.rows && n_i == 1 && p.n_h == 1 && 2 * own_rows <= NR && p.B > 1) {
        const int most = NR / own_rows, n = (p.B + most - 1) / most;
        p.bb = (p.B + n - 1) / n;
        p.n_pre = (p.B + p.bb - 1) / p.bb;
    }
    const int64_t items = (int64_t)p.B * p.n_rt + p.n_pre;
    if (items > INT32_MAX / 2) {
        set_error("latent_attention: too many query rows");
        return -1;
    }
    p.lead = lead_of(p.R);
    p.panels = p.R / 64 + 1;
    p.n_groups = p.panels > GROUP + 1 ? 2 : 1;
    p.group_bytes[0] = (p.n_groups > 1 ? GROUP : p.panels) * PANEL;
    p.group_bytes[1] = p.panels * PANEL - p.group_bytes[0];
    p.q_pitch = (p.bb ? NR : p.own_pitch) * 128;
    p.q_zero = own_rows % 16 != 0 || p.bb * own_rows % 16 != 0;
    const int fixed = p.panels * p.q_pitch + PANEL + (int)sizeof(Extra), tile = p.panels * PANEL;
    p.stages[0] = p.stages[1] = std::min(MAX_STAGES, (SMEM_MAX - fixed) / tile);
    // (what is left may hold one more first group: more loads in flight where there are few query rows)
    if (p.n_groups > 1 && p.stages[0] < MAX_STAGES && SMEM_MAX - fixed - p.stages[0] * tile >= p.group_bytes[0]) ++p.stages[0];
    const int used = fixed + p.stages[0] * p.group_bytes[0] + p.stages[1] * p.group_bytes[1];
    const int smem = std::min(SMEM_MAX, used + 1023);
    p.slack = smem - used;

    const int64_t tiles_seq = (a.c.Smax + KT - 1) / KT + (p.prefix_lens ? (p.prefix_max + KT - 1) / KT : 0);
    const int grid = (int)std::min<int64_t>(std::min(n_sm, MAX_CTAS), items * (std::max<int64_t>(tiles_seq, 1) + p.lead));

    CUtensorMap mq, mqp, mc, mcp;
    const int64_t D = p.R + p.Dr, qs[3] = {p.H, p.Lq, p.B}, qt[3] = {a.q.sh, a.q.ss, a.q.sb};
    if (!make_map(&mq, a.q.p, BF16, D, qs, qt, {p.hh, p.ii, 1})) return -1;
    mqp = mq;
    if (p.bb && !make_map(&mqp, a.q.p, BF16, D, qs, qt, {p.hh, p.ii, p.bb})) return -1;
    if (a.c.Smax > 0 && !make_map(&mc, a.c.rows, BF16, D, {a.c.Smax, a.c.B, 1}, {D, a.c.Smax * D, D}, {KT, 1, 1})) return -1;
    if (a.prefix.rows && !make_map(&mcp, a.prefix.rows, BF16, D, {a.prefix.Smax, 1, 1}, {D, D, D}, {KT, 1, 1})) return -1;
    if (a.c.Smax == 0) mc = a.prefix.rows ? mcp : mq;  // (never read: there are no own tiles)
    if (!a.prefix.rows) mcp = mc;

    // workspace: the line's data, then the parts
    p.by_item = p.bb || items <= grid;
    const int64_t slots_pre = p.bb ? p.n_pre + grid : 0, slots_own = p.bb ? (int64_t)p.B * p.n_rt + grid : 2 * (int64_t)grid;
    p.own_base = slots_pre * NR * p.R;
    const int64_t n_o = p.own_base + slots_own * p.own_pitch * p.R, n_ml = (p.bb ? items + grid : 2 * (int64_t)grid) * NR;
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    const int64_t at_joins = 256, at_ml = at_joins + up((p.by_item ? items : grid) * 16), at_o = at_ml + up(n_ml * 8);
    char* ws = nullptr;
    if (cuda_failed(cudaMallocAsync((void**)&ws, at_o + up(n_o * 4), st), "latent_attention: workspace")) return -1;
    p.n_used = (int*)ws;
    p.joins = (int4*)(ws + at_joins);
    p.part_ml = (float2*)(ws + at_ml);
    p.part_o = (float*)(ws + at_o);

    int rc = 0;
    auto kern = latent_attn_kernel<BF16>;
    static std::atomic<uint64_t> ready{0};  // devices (of the first 64) whose kernel may use this much shared memory
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(ready.load() & bit)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX), ctx)) rc = -1;
        else ready.fetch_or(bit);
    }
    if (!rc) {
        kern<<<grid, NTHREADS, smem, st>>>(mq, mqp, mc, mcp, p);
        if (cuda_failed(cudaGetLastError(), "latent_attention launch")) rc = -1;
    }
    if (!rc && (p.bb || grid > 1)) {
        cudaLaunchConfig_t cfg{};
        // 128 dims a warp (fewer instructions) where a quarter of the SMs get a block with that, else 32 (calls of 1 token, 16 heads and
        // 512 dims with 128 / 32 a warp, us: 64 sequences behind a prefix 83 / 106; without, 16 sequences, 64 blocks, 65.0 / 66.5;
        // 8, 42.7 / 39.3; one 42.0 / 23.0). Along the parts as many warps as leave each JOIN_FLIGHT of them, one step's loads (2 a
        // warp: 41.2 us instead of 39.8 for 32 sequences of 100 to 8192 rows, drafts of 5 tokens of 20 heads).
        const int64_t join_items = p.bb ? p.B : std::min<int64_t>(items, grid), row_blocks = (own_rows + JOIN_ROWS - 1) / JOIN_ROWS;
        const bool wide = join_items * row_blocks * 4 >= n_sm;
        const int dims = wide ? 128 : 32, expected = (int)(grid / (p.bb ? p.n_pre : join_items)) + 2;
        p.join_dims = wide ? (p.R + dims - 1) / dims : 1;
        p.join_groups = 1;
        while (2 * p.join_dims * p.join_groups <= JOIN_WARPS && (!wide || p.join_groups * JOIN_FLIGHT < expected)) p.join_groups *= 2;
        cfg.gridDim = dim3((unsigned)join_items, (unsigned)row_blocks, (p.R + dims * p.join_dims - 1) / (dims * p.join_dims));
        cfg.blockDim = dim3(p.join_dims * p.join_groups * 32);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        if (cuda_failed(cudaLaunchKernelEx(&cfg, wide ? latent_join_kernel<T, 4> : latent_join_kernel<T, 1>, p), "latent_attention join launch")) rc = -1;
    }
    cudaFreeAsync(ws, st);
    return rc;
}

}  // namespace

int launch_latent_attention(const LatentAttnArgs& a, cudaStream_t st) {
    if (a.c.Smax == 0 && !a.prefix.rows) {
        const int64_t rows = a.c.B * a.H * a.Lq, n = rows * a.c.R;
        latent_nothing_kernel<<<(unsigned)std::min<int64_t>(1184, (n + 255) / 256), 256, 0, st>>>((uint16_t*)a.o, n, a.lse, rows);
        return cuda_failed(cudaGetLastError(), "latent_attention launch") ? -1 : 0;
    }
    return a.c.dtype == BF16 ? launch<true>(a, st) : launch<false>(a, st);
}

}  // namespace gtb
