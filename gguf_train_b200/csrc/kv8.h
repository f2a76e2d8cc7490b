// Validated argument bundles of the block-scaled 8-bit cache calls (kv8_api.cu -> kv8_cache.cu, kv8_attn.cu)
// and of the multi-axis rotary embedding (rope_axes.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/gtb_attn.h"

namespace gtb {

// One operand (B, H, S, D) with a unit innermost stride; strides in elements
struct Rows3 {
    void* p;
    int64_t sb, sh, ss;
};

struct Kv8AppendArgs {
    gtb_kv8 c;
    Rows3 k, v;
    int dtype;
    int64_t n;
    const int32_t* counts;  // nullable
    int advance;
    int* status;
};
int launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t st);

struct Kv8ReadArgs {
    gtb_kv8 c;
    const int32_t* start;  // nullable
    int64_t n;
    void *k, *v;           // (B, Hkv, n, D) contiguous
    int dtype;
};
int launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t st);

struct Kv8EvictArgs {
    gtb_kv8 src, dst;
    const float* score;
    int64_t budget, recent;
    float* score_out;  // nullable
    int32_t* kept;
};
int launch_kv8_evict(const Kv8EvictArgs& a, cudaStream_t st);

struct Kv8AttnArgs {
    gtb_kv8 c;
    Rows3 q, o;
    int dtype;
    int64_t H, Lq;
    float scale;             // resolved (> 0)
    const int32_t* counts;   // nullable
    const float* score_in;   // both or neither
    float* score_out;
    float* lse;              // (B, H, Lq), nullable
};
int launch_kv8_attention(const Kv8AttnArgs& a, cudaStream_t st);

// Pair table of a multi-axis rotary embedding: axis of each pair and its frequency in turns per position,
// as the fraction of a turn in 64-bit fixed point
constexpr int ROPE_MAX_PAIRS = 128;
struct RopeAxesTable {
    uint64_t turn[ROPE_MAX_PAIRS];
    uint8_t axis[ROPE_MAX_PAIRS];
};
struct RopeAxesArgs {
    RopeAxesTable tab;
    Rows3 x[2], y[2];
    int64_t heads[2];  // heads of x[0], x[1]; 0: absent
    int64_t B, S;
    int D, pairs, mode, dtype;
    float sin_sign;
    const int32_t* pos;
    int64_t pos_axis, pos_batch;
};
int launch_rope_axes(const RopeAxesArgs& a, cudaStream_t st);

}  // namespace gtb
