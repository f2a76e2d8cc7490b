// The block-scaled 8-bit cache: append, read back, evict. All of it moves bytes: HBM bound, or latency bound
// for a token at a time. Work goes in chunks of 16 codes (a head size is a multiple of 16, so a chunk
// lies in one row): 16 bytes of codes against 16 values. Scale s = largest |value| / M, code = round(x / s) in IEEE
// f32 steps (kv8.cuh).

#include <algorithm>
#include <type_traits>

#include "gtb_common.cuh"
#include "kv8.cuh"

namespace gtb {
namespace {

// Row of chunk e of a block (e < 128 * 16 + 1, cpr <= 16 chunks a row): a product with ceil(2^16 / cpr), exact there
struct RowOf {
    unsigned mul;
    explicit RowOf(int64_t D) : mul((unsigned)(65536 / (D / 16) + (65536 % (D / 16) != 0))) {}
    __device__ unsigned operator()(unsigned e) const { return e * mul >> 16; }
};

// The CTA's largest x and largest y
__device__ __forceinline__ float2 block_max(float2 v, float2* red) {
    for (int o = 16; o; o >>= 1) {
        v.x = fmaxf(v.x, __shfl_xor_sync(0xffffffffu, v.x, o));
        v.y = fmaxf(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
    }
    if (blockDim.x == 32) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[threadIdx.x & 31 & ((blockDim.x >> 5) - 1)];  // blockDim a power of two
    for (int o = (int)(blockDim.x >> 6); o; o >>= 1) {
        v.x = fmaxf(v.x, __shfl_xor_sync(0xffffffffu, v.x, o));
        v.y = fmaxf(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
    }
    return v;
}

// 16 values of a row: 16-byte loads where the rows allow them
template <typename T, bool VEC>
struct Chunk {
    static constexpr int W = VEC ? (int)sizeof(T) : 16;
    using Word = typename std::conditional<VEC, uint4, T>::type;
    Word w[W];
    __device__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = ((const Word*)p)[i];
    }
    __device__ void values(int q, float* x) const {  // values 4q .. 4q + 3
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = Elem<T>::load((const T*)w + 4 * q + i);
    }
    // |x| of the largest finite value; `odd` if any is not finite
    __device__ float amax(bool& odd) const {
        float m = 0.0f;
        if constexpr (VEC && sizeof(T) == 2) {
            // the bits of |x| order as |x| does, two values a word; what is not finite comes last
            uint32_t u = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                u = __vmaxu2(u, w[i].x & 0x7fff7fffu);
                u = __vmaxu2(u, w[i].y & 0x7fff7fffu);
                u = __vmaxu2(u, w[i].z & 0x7fff7fffu);
                u = __vmaxu2(u, w[i].w & 0x7fff7fffu);
            }
            const uint32_t top = max(u & 0xffffu, u >> 16);
            if (top < (std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u)) {
                const unsigned short b = (unsigned short)top;
                return Elem<T>::load((const T*)&b);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float x[4];
            values(q, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                odd |= !(fabsf(x[i]) <= 3.402823466e38f);
                m = fmaxf(m, finite_abs(x[i]));
            }
        }
        return m;
    }
    template <int FMT>
    __device__ uint4 codes(const Quantiser& z, bool odd) const {
        uint32_t r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float x[4];
            values(q, x);
            r[q] = quantise8x4<FMT>(x, z, 1.0f, odd);
        }
        return make_uint4(r[0], r[1], r[2], r[3]);
    }
};

// 16 codes at an old scale (their values may be NaN only where a caller's own e4m3 codes are)
template <int FMT>
struct Codes16 {
    uint4 w;
    // the largest finite |value|, without the scale
    __device__ float amax(bool& odd) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        if constexpr (FMT == GTB_KV8_INT8) {
            // bytes as pairs of 16-bit integers, largest and smallest of all
            uint32_t hi = 0, lo = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t a, b;  // bytes 0, 1 and 2, 3 with their signs (a selector of 8 + i repeats byte i's)
                asm("prmt.b32 %0, %1, 0, 0x9180;" : "=r"(a) : "r"(u[q]));
                asm("prmt.b32 %0, %1, 0, 0xb3a2;" : "=r"(b) : "r"(u[q]));
                hi = __vimax3_s16x2(hi, a, b);
                lo = __vimin3_s16x2(lo, a, b);
            }
            const int top = max((int)(int16_t)(hi & 0xffff), (int)(int16_t)(hi >> 16));
            const int bot = min((int)(int16_t)(lo & 0xffff), (int)(int16_t)(lo >> 16));
            odd |= bot < -127;  // a code that no quantiser gives, and that has to saturate
            return (float)max(top, -bot);
        } else {
            // magnitudes order as their bits; 0x7f is NaN
            uint32_t m = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) m = __vmaxu2(m, __vmaxu2(u[q] & 0x007f007fu, (u[q] >> 8) & 0x007f007fu));
            const uint32_t top = max(m & 0xffffu, m >> 16);
            if (top < 0x7fu) return Code8<FMT>::value((uint8_t)top);
            odd = true;
            float f = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float x[4];
                values8x4<FMT>(u[q], x);
#pragma unroll
                for (int i = 0; i < 4; ++i) f = fmaxf(f, finite_abs(x[i]));
            }
            return f;
        }
    }
    // codes of (code * s_old) / s; z: of s, its factors times s_old
    __device__ uint4 again(float s_old, const Quantiser& z, bool odd) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        uint32_t r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float x[4];
            values8x4<FMT>(u[q], x);
            r[q] = quantise8x4<FMT>(x, z, s_old, odd);
        }
        return make_uint4(r[0], r[1], r[2], r[3]);
    }
};

// One CTA per (touched block, sequence x kv head), K and V together. The new rows stay in registers between the largest
// value and the codes (KEEP chunks of each a thread; what does not fit is read again, from L2). 8 sequences, up to 4099
// tokens, 8 heads of 128, f16 to e4m3 blocks of 32: 31 us for 110 MB (3.6 TB/s), bound by the conversions' issue slots (70 %
// busy); with 2 / 4 chunks kept the append and a read of it take 75 / 86 us (fewer threads a block hide less).
template <typename T, int FMT, bool VEC, int KEEP>
__global__ void __launch_bounds__(256) kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a, unsigned blocks, RowOf row_of) {
    __shared__ float2 red[8];
    const gtb_kv8& c = a.c;
    const unsigned bhx = blockIdx.x / blocks, jx = blockIdx.x - bhx * blocks;
    const int64_t bh = bhx, b = bhx / (unsigned)c.Hkv, hk = bh - b * c.Hkv;
    const int bt = c.block;
    const int pos = (int)clamp64(c.lens[b], 0, c.Smax);
    const int cnt = a.counts ? (int)clamp64(a.counts[b], 0, a.n) : (int)a.n;
    const int end = (int)min((int64_t)pos + cnt, c.Smax);
    if ((int64_t)pos + cnt > c.Smax && jx == 0 && threadIdx.x == 0) atomicCAS(a.status, 0, 61);
    const int shift = 31 - __clz(bt), j = (pos >> shift) + (int)jx;
    const int r0 = max(j * bt, pos), r1 = (int)min((int64_t)(j + 1) * bt, (int64_t)end);  // new rows of this block
    if (r0 >= r1) return;
    const unsigned cpr = (unsigned)c.D / 16, n_new = (unsigned)(r1 - r0) * cpr;
    const T* src_k = (const T*)a.k.p + b * a.k.sb + hk * a.k.sh + (int64_t)(r0 - pos) * a.k.ss;
    const T* src_v = (const T*)a.v.p + b * a.v.sb + hk * a.v.sh + (int64_t)(r0 - pos) * a.v.ss;
    const int64_t at = (bh * c.Smax + (int64_t)j * bt) * c.D, sat = bh * ((c.Smax + bt - 1) >> shift) + j;
    const bool had = j * bt < pos;
    const float2 s_old = had ? make_float2(c.k_scale[sat], c.v_scale[sat]) : make_float2(0.0f, 0.0f);
    Chunk<T, VEC> kk[KEEP], kv[KEEP];
    float2 m = make_float2(0.0f, 0.0f);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const unsigned e = threadIdx.x + i * blockDim.x, r = row_of(e), d = (e - r * cpr) * 16;
        if (e < n_new) {
            kk[i].load(src_k + r * a.k.ss + d);
            kv[i].load(src_v + r * a.v.ss + d);
        }
    }
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
        if (threadIdx.x + i * blockDim.x < n_new) {
            m.x = fmaxf(m.x, kk[i].amax(odd));
            m.y = fmaxf(m.y, kv[i].amax(odd));
        }
#pragma unroll 1
    for (unsigned e = threadIdx.x + KEEP * blockDim.x; e < n_new; e += blockDim.x) {
        const unsigned r = row_of(e), d = (e - r * cpr) * 16;
        Chunk<T, VEC> t;
        t.load(src_k + r * a.k.ss + d);
        m.x = fmaxf(m.x, t.amax(odd));
        t.load(src_v + r * a.v.ss + d);
        m.y = fmaxf(m.y, t.amax(odd));
    }
    m = block_max(m, red);
    const float2 s = make_float2(fmaxf(s_old.x, scale_of<FMT>(m.x)), fmaxf(s_old.y, scale_of<FMT>(m.y)));
    const Quantiser zk(s.x), zv(s.y);
    // the rows already held, where their scale grew
    auto requantise = [&](void* codes, float from, const Quantiser& z) {
        Quantiser zo = z;
        zo.times(from);
        uint4* held = (uint4*)((uint8_t*)codes + at);
        const unsigned n_old = (unsigned)(r0 - j * bt) * cpr;
#pragma unroll 1
        for (unsigned e = threadIdx.x; e < n_old; e += blockDim.x) {
            const Codes16<FMT> w{held[e]};
            bool nan = false;
            w.amax(nan);
            held[e] = w.again(from, zo, nan);
        }
    };
    if (had && s.x > s_old.x) requantise(c.k, s_old.x, zk);
    if (had && s.y > s_old.y) requantise(c.v, s_old.y, zv);
    const int64_t to = at + (int64_t)(r0 - j * bt) * c.D;
    uint4 *dst_k = (uint4*)((uint8_t*)c.k + to), *dst_v = (uint4*)((uint8_t*)c.v + to);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const unsigned e = threadIdx.x + i * blockDim.x;
        if (e < n_new) {
            dst_k[e] = kk[i].template codes<FMT>(zk, odd);
            dst_v[e] = kv[i].template codes<FMT>(zv, odd);
        }
    }
#pragma unroll 1
    for (unsigned e = threadIdx.x + KEEP * blockDim.x; e < n_new; e += blockDim.x) {
        const unsigned r = row_of(e), d = (e - r * cpr) * 16;
        Chunk<T, VEC> t;
        t.load(src_k + r * a.k.ss + d);
        dst_k[e] = t.template codes<FMT>(zk, odd);
        t.load(src_v + r * a.v.ss + d);
        dst_v[e] = t.template codes<FMT>(zv, odd);
    }
    if (threadIdx.x == 0) {
        c.k_scale[sat] = s.x;
        c.v_scale[sat] = s.y;
    }
}

__global__ void kv8_advance_kernel(const Kv8AppendArgs a) {
    const int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= a.c.B) return;
    const int64_t pos = clamp64(a.c.lens[b], 0, a.c.Smax);
    const int64_t cnt = a.counts ? clamp64(a.counts[b], 0, a.n) : a.n;
    a.c.lens[b] = (int32_t)min(pos + cnt, a.c.Smax);
}

// A thread reads chunks of READ_ROWS rows of one (sequence, kv head, K or V) and writes their values. HBM bound: the
// read after the append above 39 us (5.2 TB/s), 16 x 4096 tokens x 8 heads of 128 to bf16 72 us (5.6 TB/s).
constexpr int READ_ROWS = 4;
template <typename T, int FMT>
__global__ void __launch_bounds__(256) kv8_read_kernel(const __grid_constant__ Kv8ReadArgs a) {
    const gtb_kv8& c = a.c;
    const unsigned cpr = (unsigned)c.D / 16, rows = 256 / cpr;  // rows a CTA covers at a time
    const unsigned row = threadIdx.x / cpr, chunk = threadIdx.x - row * cpr;
    if (row >= rows) return;
    const int shift = 31 - __clz(c.block);
    const int64_t nb = (c.Smax + c.block - 1) >> shift;
    for (int64_t p = blockIdx.y; p < 2 * c.B * c.Hkv; p += gridDim.y) {
        const bool is_v = p >= c.B * c.Hkv;
        const int64_t bh = is_v ? p - c.B * c.Hkv : p;
        const int64_t start = a.start ? a.start[bh / c.Hkv] : 0;
        const uint4* codes = (const uint4*)(is_v ? c.v : c.k) + bh * c.Smax * cpr + chunk;
        const float* scale = (is_v ? c.v_scale : c.k_scale) + bh * nb;
        T* out = (T*)(is_v ? a.v : a.k) + bh * a.n * c.D + chunk * 16;
        uint4 w[READ_ROWS];
        float s[READ_ROWS];
        const int64_t t0 = (int64_t)blockIdx.x * (rows * READ_ROWS) + row;
#pragma unroll
        for (int i = 0; i < READ_ROWS; ++i) {
            const int64_t t = t0 + i * rows, r = start + t;
            const bool live = t < a.n && r >= 0 && r < c.Smax;
            w[i] = live ? codes[r * cpr] : make_uint4(0, 0, 0, 0);
            s[i] = live ? scale[r >> shift] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < READ_ROWS; ++i) {
            const int64_t t = t0 + i * rows;
            if (t >= a.n) break;
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            __align__(16) T y[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float x[4];
                values8x4<FMT>(u[q], x);
#pragma unroll
                for (int k = 0; k < 4; ++k) Elem<T>::store(y + 4 * q + k, __fmul_rn(x[k], s[i]));
            }
#pragma unroll
            for (int k = 0; k < (int)sizeof(T); ++k) ((uint4*)(out + t * c.D))[k] = ((const uint4*)y)[k];
        }
    }
}

// ------------------------------------------------------------------ eviction

// Order of scores as unsigned integers: larger score, larger key; NaN as -inf, -0 as 0
__device__ __forceinline__ uint32_t score_key(float s) {
    if (!(s == s)) s = -INFINITY;
    const uint32_t u = __float_as_uint(__fadd_rn(s, 0.0f));
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int SEL_THREADS = 1024, SEL_WARPS = SEL_THREADS / 32, SEL_KEEP = 16, SEL_TILE = SEL_THREADS * SEL_KEEP;
constexpr int SEL_BINS = 2048;

// Sum over the warps before this one and over all, of one packed value per warp
__device__ __forceinline__ uint64_t warps_before(uint64_t v, uint64_t* sh, uint64_t& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (lane == 0) sh[w] = v;
    __syncthreads();
    uint64_t x = sh[lane], s = x;
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    total = __shfl_sync(0xffffffffu, s, 31);
    const uint64_t r = __shfl_sync(0xffffffffu, s - x, w);
    __syncthreads();
    return r;
}

// Which rows stay: one CTA per (sequence, kv head). The k-th largest key among the candidates is found by
// digits of 11, 11 and 10 bits: a histogram of the keys that match so far, summed from the top. The first
// digit holds the exponent and two bits of the mantissa, which spreads the atomics. Then one sweep in row
// order takes every larger key and the first `need` that equal it. The first SEL_TILE scores stay in
// registers (warp w holds 512 consecutive ones); longer rows read theirs again each pass, from L2. 128 heads of up to
// 16k scores 15 us: three passes' latency and shared-memory atomics, with one CTA of 1024 threads an SM.
__global__ void __launch_bounds__(SEL_THREADS) kv8_select_kernel(const __grid_constant__ Kv8EvictArgs a) {
    __shared__ uint32_t hist[SEL_BINS];
    __shared__ uint64_t sh[SEL_WARPS];
    __shared__ uint32_t found[2];
    cudaTriggerProgrammaticLaunchCompletion();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t bh = blockIdx.x, b = bh / a.src.Hkv;
    const int len = (int)clamp64(a.src.lens[b], 0, a.src.Smax);
    const int budget = (int)min(a.budget, (int64_t)1 << 30), recent = (int)min(a.recent, (int64_t)1 << 30);
    const int newlen = min(len, budget);
    int32_t* kept = a.kept + bh * a.budget;
    const float* score = a.score + bh * a.src.Smax;
    for (int64_t j = newlen + threadIdx.x; j < a.budget; j += SEL_THREADS) kept[j] = -1;
    if (bh - b * a.src.Hkv == 0 && threadIdx.x == 0) a.dst.lens[b] = newlen;
    if (len <= budget) {
        for (int j = threadIdx.x; j < len; j += SEL_THREADS) kept[j] = j;
        return;
    }
    const int n = len - recent, k = budget - recent;  // n > k
    for (int j = threadIdx.x; j < recent; j += SEL_THREADS) kept[k + j] = n + j;
    if (k == 0) return;
    const int base = warp * (32 * SEL_KEEP) + lane;
    uint32_t mine[SEL_KEEP];
#pragma unroll
    for (int i = 0; i < SEL_KEEP; ++i) mine[i] = base + i * 32 < n ? score_key(score[base + i * 32]) : 0u;
    uint32_t prefix = 0, need = (uint32_t)k;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
        const uint32_t digit = pass == 2 ? 1023u : 2047u;
        for (int i = threadIdx.x; i < SEL_BINS; i += SEL_THREADS) hist[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SEL_KEEP; ++i)
            if (base + i * 32 < n && (mine[i] & mask) == prefix) atomicAdd(&hist[(mine[i] >> shift) & digit], 1u);
        for (int i = SEL_TILE + threadIdx.x; i < n; i += SEL_THREADS) {
            const uint32_t key = score_key(score[i]);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & digit], 1u);
        }
        __syncthreads();
        // thread t takes bins 2047 - 2t and 2046 - 2t: the counts above them, from the top
        const uint32_t c0 = hist[SEL_BINS - 1 - 2 * threadIdx.x], c1 = hist[SEL_BINS - 2 - 2 * threadIdx.x];
        uint32_t s = c0 + c1;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        uint64_t total;
        const uint32_t above = (uint32_t)warps_before(__shfl_sync(0xffffffffu, s, 31), sh, total) + s - c0 - c1;
        if (above < need && above + c0 >= need) {
            found[0] = SEL_BINS - 1 - 2 * threadIdx.x;
            found[1] = need - above;
        } else if (above + c0 < need && above + c0 + c1 >= need) {
            found[0] = SEL_BINS - 2 - 2 * threadIdx.x;
            found[1] = need - above - c0;
        }
        __syncthreads();
        prefix |= found[0] << shift;
        need = found[1];
        __syncthreads();
    }
    // keys above the k-th, and the first `need` equal to it, in row order; counts packed (above << 32 | equal)
    uint64_t done = 0;
    for (int t0 = 0; t0 < n; t0 += SEL_TILE) {
        if (t0 > 0) {
#pragma unroll
            for (int i = 0; i < SEL_KEEP; ++i) {
                const int e = t0 + base + i * 32;
                mine[i] = e < n ? score_key(score[e]) : 0u;
            }
        }
        uint64_t own = 0;
        uint32_t gt[SEL_KEEP], eq[SEL_KEEP];
#pragma unroll
        for (int i = 0; i < SEL_KEEP; ++i) {
            const bool in = t0 + base + i * 32 < n;
            gt[i] = __ballot_sync(0xffffffffu, in && mine[i] > prefix);
            eq[i] = __ballot_sync(0xffffffffu, in && mine[i] == prefix);
            own += ((uint64_t)__popc(gt[i]) << 32) | (uint64_t)__popc(eq[i]);
        }
        uint64_t total;
        uint64_t at = done + warps_before(own, sh, total);
        const uint32_t below = (1u << lane) - 1u;
#pragma unroll
        for (int i = 0; i < SEL_KEEP; ++i) {
            const uint32_t g = (uint32_t)(at >> 32) + __popc(gt[i] & below), e = (uint32_t)at + __popc(eq[i] & below);
            if ((gt[i] >> lane & 1u) || ((eq[i] >> lane & 1u) && e < need)) kept[g + min(e, need)] = t0 + base + i * 32;
            at += ((uint64_t)__popc(gt[i]) << 32) | (uint64_t)__popc(eq[i]);
        }
        done += total;
    }
}

// One CTA per (destination block, sequence x kv head), K and V together: the kept rows' values, their largest, the new
// scale, the new codes. As in the append, KEEP chunks of each a thread stay in registers. 16 sequences to 4096 rows,
// 8 heads of 128: 93 us, bound by the conversions (ALU 65 %, issue slots 69 % busy) rather than by its 0.27 GB (41 us).
template <int FMT, int KEEP>
__global__ void __launch_bounds__(256) kv8_gather_kernel(const __grid_constant__ Kv8EvictArgs a, unsigned blocks, RowOf row_of) {
    __shared__ float2 red[8];
    cudaGridDependencySynchronize();  // the kept rows and the new lengths are there
    const unsigned bhx = blockIdx.x / blocks, j = blockIdx.x - bhx * blocks;
    const int64_t bh = bhx;
    const int bs = a.src.block, bd = a.dst.block, shift = 31 - __clz(bs);
    const int newlen = a.dst.lens[bhx / (unsigned)a.src.Hkv];
    const int r0 = (int)(j * bd), r1 = min(r0 + bd, newlen);
    const int32_t* kept = a.kept + bh * a.budget + r0;
    if (a.score_out)
        for (int64_t r = r0 + threadIdx.x; r < min((int64_t)r0 + bd, a.dst.Smax); r += blockDim.x)
            a.score_out[bh * a.dst.Smax + r] = r < newlen ? a.score[bh * a.src.Smax + kept[r - r0]] : 0.0f;
    if (r0 >= r1) return;
    const unsigned cpr = (unsigned)a.src.D / 16, n = (unsigned)(r1 - r0) * cpr;
    const uint4 *src_k = (const uint4*)a.src.k + bh * a.src.Smax * cpr, *src_v = (const uint4*)a.src.v + bh * a.src.Smax * cpr;
    const int64_t ns = bh * ((a.src.Smax + bs - 1) >> shift), to = (bh * a.dst.Smax + r0) * cpr;
    const float *sk = a.src.k_scale + ns, *sv = a.src.v_scale + ns;
    uint4 *dst_k = (uint4*)a.dst.k + to, *dst_v = (uint4*)a.dst.v + to;
    Codes16<FMT> wk[KEEP], wv[KEEP];
    float2 s_old[KEEP], m = make_float2(0.0f, 0.0f);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const unsigned e = threadIdx.x + i * blockDim.x, r = row_of(e);
        s_old[i] = make_float2(0.0f, 0.0f);
        if (e < n) {
            const unsigned row = kept[r];
            const int64_t at = (int64_t)row * cpr + (e - r * cpr);
            wk[i].w = src_k[at];
            wv[i].w = src_v[at];
            s_old[i] = make_float2(sk[row >> shift], sv[row >> shift]);
        }
    }
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
        if (threadIdx.x + i * blockDim.x < n) {
            m.x = fmaxf(m.x, finite_abs(__fmul_rn(wk[i].amax(odd), s_old[i].x)));
            m.y = fmaxf(m.y, finite_abs(__fmul_rn(wv[i].amax(odd), s_old[i].y)));
        }
#pragma unroll 1
    for (unsigned e = threadIdx.x + KEEP * blockDim.x; e < n; e += blockDim.x) {
        const unsigned r = row_of(e), row = kept[r];
        const int64_t at = (int64_t)row * cpr + (e - r * cpr);
        m.x = fmaxf(m.x, finite_abs(__fmul_rn(Codes16<FMT>{src_k[at]}.amax(odd), sk[row >> shift])));
        m.y = fmaxf(m.y, finite_abs(__fmul_rn(Codes16<FMT>{src_v[at]}.amax(odd), sv[row >> shift])));
    }
    m = block_max(m, red);
    const float2 s = make_float2(scale_of<FMT>(m.x), scale_of<FMT>(m.y));
    const Quantiser zk(s.x), zv(s.y);
    auto again = [&](const Codes16<FMT>& w, float from, const Quantiser& z) {
        Quantiser zo = z;
        zo.times(from);
        return w.again(from, zo, odd);
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const unsigned e = threadIdx.x + i * blockDim.x;
        if (e < n) {
            dst_k[e] = again(wk[i], s_old[i].x, zk);
            dst_v[e] = again(wv[i], s_old[i].y, zv);
        }
    }
#pragma unroll 1
    for (unsigned e = threadIdx.x + KEEP * blockDim.x; e < n; e += blockDim.x) {
        const unsigned r = row_of(e), row = kept[r];
        const int64_t at = (int64_t)row * cpr + (e - r * cpr);
        dst_k[e] = again(Codes16<FMT>{src_k[at]}, sk[row >> shift], zk);
        dst_v[e] = again(Codes16<FMT>{src_v[at]}, sv[row >> shift], zv);
    }
    if (threadIdx.x == 0) {
        const int64_t nd = bh * ((a.dst.Smax + bd - 1) >> (31 - __clz(bd))) + j;
        a.dst.k_scale[nd] = s.x;
        a.dst.v_scale[nd] = s.y;
    }
}

// Chunks of each of K and V a thread keeps. Eviction of 16 x 16k tokens to 4k with 2 / 4 / 8: 183 / 183 / 207 us at blocks of
// 64 tokens, 181 / 193 / 224 us at 16 (fewer threads a block)
constexpr int GATHER_KEEP = 2;

// Threads for `chunks` of work in a CTA: a power of two, `each` chunks a thread where there are enough
int threads_for(int64_t chunks, int each) {
    int t = 32;
    while (t < 256 && t * each < chunks) t *= 2;
    return t;
}

bool grid_fits(int64_t n, const char* ctx) {
    if (n <= INT32_MAX) return true;
    set_errorf("%s: batch x kv heads x blocks must fit in int32", ctx);
    return false;
}

template <typename T, int FMT>
int append_t(const Kv8AppendArgs& a, cudaStream_t st) {
    // a block beyond the capacity is never touched
    const int64_t blocks = std::min((a.n + a.c.block - 2) / a.c.block + 1, (a.c.Smax + a.c.block - 1) / a.c.block + 1);
    const int64_t n = blocks * a.c.B * a.c.Hkv;
    if (!grid_fits(n, "kv8_append")) return -1;
    constexpr int N = 16 / sizeof(T);
    bool vec = true;
    for (const Rows3* r : {&a.k, &a.v})
        vec = vec && ((uintptr_t)r->p & 15) == 0 && r->sb % N == 0 && r->sh % N == 0 && r->ss % N == 0;
    const int threads = threads_for(std::min<int64_t>(a.n, a.c.block) * (a.c.D / 16), 2);
    const dim3 grid((unsigned)n);
    auto go = [&](auto kern) { kern<<<grid, threads, 0, st>>>(a, (unsigned)blocks, RowOf(a.c.D)); };
    if (!vec) go(kv8_append_kernel<T, FMT, false, 1>);
    else go(kv8_append_kernel<T, FMT, true, sizeof(T) == 4 ? 1 : 2>);
    return cuda_failed(cudaGetLastError(), "kv8_append launch") ? -1 : 0;
}

template <int FMT>
int append_fmt(const Kv8AppendArgs& a, cudaStream_t st) {
    switch (a.dtype) {
        case F32: return append_t<float, FMT>(a, st);
        case F16: return append_t<__half, FMT>(a, st);
        default: return append_t<__nv_bfloat16, FMT>(a, st);
    }
}

template <int FMT>
int read_fmt(const Kv8ReadArgs& a, cudaStream_t st) {
    const int64_t rows = 256 / (a.c.D / 16) * READ_ROWS;
    const dim3 grid((unsigned)((a.n + rows - 1) / rows), (unsigned)std::min<int64_t>(2 * a.c.B * a.c.Hkv, 65535));
    switch (a.dtype) {
        case F32: kv8_read_kernel<float, FMT><<<grid, 256, 0, st>>>(a); break;
        case F16: kv8_read_kernel<__half, FMT><<<grid, 256, 0, st>>>(a); break;
        default: kv8_read_kernel<__nv_bfloat16, FMT><<<grid, 256, 0, st>>>(a); break;
    }
    return cuda_failed(cudaGetLastError(), "kv8_read launch") ? -1 : 0;
}

template <int FMT>
bool gather(const Kv8EvictArgs& a, cudaStream_t st) {
    // score_out covers dst.Smax rows, the codes only the budget
    const int64_t rows = a.score_out ? a.dst.Smax : a.budget;
    const int64_t blocks = (rows + a.dst.block - 1) / a.dst.block, n = blocks * a.src.B * a.src.Hkv;
    if (!grid_fits(n, "kv8_evict")) return false;
    const int64_t chunks = std::min<int64_t>(a.budget, a.dst.block) * (a.src.D / 16);
    const int threads = threads_for(chunks, GATHER_KEEP);
    return launch_behind("kv8_evict: gather launch", kv8_gather_kernel<FMT, GATHER_KEEP>, dim3((unsigned)n),
                         threads, st, 0, a, (unsigned)blocks, RowOf(a.src.D));
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
    kv8_select_kernel<<<(unsigned)(a.src.B * a.src.Hkv), SEL_THREADS, 0, st>>>(a);
    if (cuda_failed(cudaGetLastError(), "kv8_evict: select launch")) return -1;
    return (a.src.format == GTB_KV8_INT8 ? gather<GTB_KV8_INT8>(a, st) : gather<GTB_KV8_E4M3>(a, st)) ? 0 : -1;
}

}  // namespace gtb
