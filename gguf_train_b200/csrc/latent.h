// Validated argument bundles of the latent attention calls (latent_api.cu -> latent_cache.cu, latent_attn_sm100.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/gtb_attn.h"
#include "kv8.h"

namespace gtb {

struct LatentAppendArgs {
    gtb_latent c;
    Rows3 latent, k_rope;    // strides of batch, -, token
    int dtype;               // of both
    int64_t n;
    const int32_t* counts;   // nullable
    const int32_t* offset;   // nullable: rows of a shared prefix, added to the positions
    bool turns;              // k_rope is rotated by `tab`
    int mode;
    RopeAxesTable tab;
    int advance;
    int* status;
};
int launch_latent_append(const LatentAppendArgs& a, cudaStream_t st);

struct LatentAttnArgs {
    gtb_latent c;
    gtb_latent prefix;       // rows null: none
    Rows3 q;
    void* o;                 // (B, H, Lq, R) contiguous
    int64_t H, Lq;
    float scale;
    const int32_t* counts;   // nullable
    float* lse;              // (B, H, Lq), nullable
    int* status;
};
int launch_latent_attention(const LatentAttnArgs& a, cudaStream_t st);

}  // namespace gtb
