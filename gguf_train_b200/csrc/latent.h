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

// Expanded latent attention: q, o, lse, g, dq (B, H, L, .), k, v, dk, dv (B, Hkv, S, .), the rotary keys and their gradient (B, 1, S, Dr)
struct LatentSdpaArgs {
    int64_t B, H, Hkv, L, S;
    int Dn, Dr;              // Dv = Dn
    gtb_tensor4 q, k, k_rope, v, o;
    float* lse;              // (B, H, L); the forward's may be null
    const int32_t* lens;     // nullable
    float scale;
    int causal;
    gtb_tensor4 g, dq, dk, dk_rope, dv;  // backward only
    int* status;
};
int launch_latent_sdpa_fwd(const LatentSdpaArgs& a, cudaStream_t st);
int launch_latent_sdpa_bwd(const LatentSdpaArgs& a, cudaStream_t st);

// tokens of sequence b that take part
__device__ __forceinline__ int latent_tokens(const int32_t* lens, int b, int64_t n) {
    return lens ? (int)min((int64_t)max(lens[b], 0), n) : (int)n;
}

}  // namespace gtb
