// Rotary position embedding with several position axes, of one tensor or of q and k in one launch.
// The angle of pair i of token (b, s) is pos[axis(i)][b][s] * f(i). Its value modulo a turn is all that the
// sine and cosine see, so the frequency is kept as turns per position in 64-bit fixed point: the integer
// product position * turn modulo 2^64 drops the whole turns exactly, and what is left is right to 2^-31 of a turn at any
// int32 position. It becomes f32 (half a turn at most: to 2^-26) for sine and cosine.
//
// HBM bound: every value is read and written once. A CTA takes TOK tokens of one sequence and a share of the
// heads: it forms the tokens' (cos, sin) table once in shared memory, then each thread keeps the part of the table
// that belongs to its 16 bytes of a row in registers and walks the heads with 16-byte accesses, two rows in
// flight. Measured: 8 x 4096 tokens, 32 + 8 heads of 128, bf16 115 us, 5.8 TB/s (166 with one row in flight and three CTAs
// an SM); 6 x 2047 tokens, 16 + 16 heads of 80, f32 43 us, 5.9 TB/s; one token of 64 sequences is a launch, 4 us.

#include <algorithm>

#include "gtb_common.cuh"
#include "kv8.h"

namespace gtb {
namespace {

// (cos, sin) of a pair at position p
__device__ __forceinline__ float2 turn_of(int32_t p, uint64_t turn, float sin_sign) {
    const int32_t frac = (int32_t)(((uint64_t)(int64_t)p * turn) >> 32);  // signed fraction of a turn, 2^-32
    float s, c;
    sincospif((float)frac * 4.656612873077393e-10f, &s, &c);  // x 2 * 2^-32
    return make_float2(c, s * sin_sign);
}

template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};

constexpr int THREADS = 256, FLIGHT = 2;

// A thread owns one piece of a row: V values, and in mode 2 their V partners P further on (V = 16 bytes, or one
// value where sizes, strides or alignment allow no more). Pieces per row: the rotated ones first, then the
// dims that pass through.
template <typename T, int V, int MODE>
__global__ void __launch_bounds__(THREADS, 4) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a, int tok, int rot, int pieces,
                                                            int groups, int heads_per_group) {
    extern __shared__ float2 tab[];  // [tok][pairs]
    const int64_t s0 = (int64_t)blockIdx.x * tok, b = blockIdx.z;
    const int P = a.pairs;
    // (a parameter indexed by lane is read a lane at a time, so each pair's frequency and axis are read once: read at
    // every entry of the table, those reads were 45 us of the 8 x 4096 tokens)
    __shared__ uint64_t turn[ROPE_MAX_PAIRS];
    __shared__ int64_t axis[ROPE_MAX_PAIRS];
    if (threadIdx.x < P) {
        turn[threadIdx.x] = a.tab.turn[threadIdx.x];
        axis[threadIdx.x] = a.tab.axis[threadIdx.x] * a.pos_axis + b * a.pos_batch + s0;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < tok * P; e += THREADS) {
        const int sl = e / P, i = e - sl * P;
        if (s0 + sl < a.S) tab[e] = turn_of(a.pos[axis[i] + sl], turn[i], a.sin_sign);
    }
    __syncthreads();
    // thread -> (head group within the CTA, token, piece)
    const int per = tok * pieces;
    for (int e = threadIdx.x; e < groups * per; e += THREADS) {
        const int grp = e / per, rest = e - grp * per, sl = rest / pieces, piece = rest - sl * pieces;
        const int64_t s = s0 + sl;
        if (s >= a.S) continue;
        const int64_t all = a.heads[0] + a.heads[1];
        const int64_t h0 = ((int64_t)blockIdx.y * groups + grp) * heads_per_group, h1 = min(all, h0 + heads_per_group);
        const bool turns = piece < rot;
        const int d = turns ? piece * V : 2 * P + (piece - rot) * V;  // first value of the piece
        constexpr int NP = MODE == 2 ? V : (V + 1) / 2;  // pairs of a piece; with V = 1 and mode 0 a piece is a pair
        float2 cs[NP];
        if (turns) {
#pragma unroll
            for (int k = 0; k < NP; ++k) cs[k] = tab[sl * P + (MODE == 2 ? d + k : V == 1 ? piece : d / 2 + k)];
        }
        for (int64_t h = h0; h < h1; h += FLIGHT) {
            __align__(16) T u[FLIGHT][V];
            __align__(16) T w[FLIGHT][V];
            int64_t yo[FLIGHT];
            T* yp[FLIGHT];
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                if (h + f >= h1) break;
                const int side = h + f >= a.heads[0];
                const int64_t hh = h + f - (side ? a.heads[0] : 0);
                const T* x = (const T*)a.x[side].p + b * a.x[side].sb + hh * a.x[side].sh + s * a.x[side].ss;
                yp[f] = (T*)a.y[side].p;
                yo[f] = b * a.y[side].sb + hh * a.y[side].sh + s * a.y[side].ss;
                if constexpr (V == 1) {
                    const int c0 = !turns ? d : MODE == 2 ? d : 2 * piece;
                    u[f][0] = x[c0];
                    if (turns) w[f][0] = x[MODE == 2 ? d + P : c0 + 1];
                } else {
                    *(uint4*)u[f] = *(const uint4*)(x + d);
                    if (MODE == 2 && turns) *(uint4*)w[f] = *(const uint4*)(x + d + P);
                }
            }
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                if (h + f >= h1) break;
                T* y = yp[f] + yo[f];
                if (!turns) {
                    if constexpr (V == 1) y[d] = u[f][0];
                    else *(uint4*)(y + d) = *(const uint4*)u[f];
                    continue;
                }
                if constexpr (MODE == 2 || V == 1) {
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float x0 = Elem<T>::load(&u[f][k]), x1 = Elem<T>::load(&w[f][k]);
                        Elem<T>::store(&u[f][k], x0 * cs[k].x - x1 * cs[k].y);
                        Elem<T>::store(&w[f][k], x0 * cs[k].y + x1 * cs[k].x);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
                        const float x0 = Elem<T>::load(&u[f][2 * k]), x1 = Elem<T>::load(&u[f][2 * k + 1]);
                        Elem<T>::store(&u[f][2 * k], x0 * cs[k].x - x1 * cs[k].y);
                        Elem<T>::store(&u[f][2 * k + 1], x0 * cs[k].y + x1 * cs[k].x);
                    }
                }
                if constexpr (V == 1) {
                    const int c0 = MODE == 2 ? d : 2 * piece;
                    y[c0] = u[f][0];
                    y[MODE == 2 ? d + P : c0 + 1] = w[f][0];
                } else {
                    *(uint4*)(y + d) = *(const uint4*)u[f];
                    if (MODE == 2) *(uint4*)(y + d + P) = *(const uint4*)w[f];
                }
            }
        }
    }
}

template <typename T, int V, int MODE>
int launch(const RopeAxesArgs& a, cudaStream_t st) {
    int dev = 0, n_sm = 0;
    if (cuda_failed(cudaGetDevice(&dev), "rope_axes") ||
        cuda_failed(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev), "rope_axes"))
        return -1;
    const int64_t heads = a.heads[0] + a.heads[1];
    const int rot = V == 1 ? a.pairs : MODE == 2 ? a.pairs / V : 2 * a.pairs / V;
    const int pieces = rot + (a.D - 2 * a.pairs) / V;
    // tokens per CTA: as many as give each thread one piece of one head group, fewer for short sequences
    int tok = std::max(1, THREADS / pieces);
    tok = (int)std::min<int64_t>(tok, a.S);
    int groups = std::max(1, THREADS / (tok * pieces));  // head groups side by side in the CTA
    const int64_t blocks = (a.S + tok - 1) / tok * a.B;
    // enough CTAs for 8 per SM, but no fewer than FLIGHT heads a thread
    int64_t split = std::max<int64_t>(1, std::min<int64_t>((heads + groups * FLIGHT - 1) / (groups * FLIGHT), (n_sm * 8 + blocks - 1) / blocks));
    int64_t hpg = (heads + groups * split - 1) / (groups * split);
    split = (heads + groups * hpg - 1) / (groups * hpg);
    const size_t smem = sizeof(float2) * tok * a.pairs;
    for (int64_t b0 = 0; b0 < a.B; b0 += 65535) {
        RopeAxesArgs z = a;
        const int64_t nb = std::min<int64_t>(65535, a.B - b0);
        for (int w = 0; w < 2; ++w) {
            z.x[w].p = (T*)a.x[w].p + b0 * a.x[w].sb;
            z.y[w].p = (T*)a.y[w].p + b0 * a.y[w].sb;
        }
        z.pos = a.pos + b0 * a.pos_batch;
        const dim3 grid((unsigned)((a.S + tok - 1) / tok), (unsigned)split, (unsigned)nb);
        rope_axes_kernel<T, V, MODE><<<grid, THREADS, smem, st>>>(z, tok, rot, pieces, groups, (int)hpg);
        if (cuda_failed(cudaGetLastError(), "rope_axes launch")) return -1;
    }
    return 0;
}

// 16-byte pieces where every row, and in mode 2 its second half, starts on 16 bytes; else a value or pair a thread
// (8 x 4096 tokens as above, 120 / 333 us a call)
template <typename T>
int launch_t(const RopeAxesArgs& a, cudaStream_t st) {
    constexpr int N = 16 / sizeof(T);
    bool vec = a.D % N == 0 && (a.mode == 2 ? a.pairs % N == 0 : 2 * a.pairs % N == 0);
    for (int w = 0; w < 2; ++w) {
        if (a.heads[w] == 0) continue;
        for (const Rows3* r : {&a.x[w], &a.y[w]})
            vec = vec && ((uintptr_t)r->p & 15) == 0 && r->sb % N == 0 && r->sh % N == 0 && r->ss % N == 0;
    }
    if (a.mode == 2) return vec ? launch<T, N, 2>(a, st) : launch<T, 1, 2>(a, st);
    return vec ? launch<T, N, 0>(a, st) : launch<T, 1, 0>(a, st);
}

}  // namespace

int launch_rope_axes(const RopeAxesArgs& a, cudaStream_t st) {
    switch (a.dtype) {
        case F32: return launch_t<float>(a, st);
        case F16: return launch_t<__half>(a, st);
        default: return launch_t<__nv_bfloat16>(a, st);
    }
}

}  // namespace gtb
