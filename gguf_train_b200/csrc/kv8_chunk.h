// The tcgen05 paths of kv8_attention for many query rows (kv8_chunk_sm100.cu, kv8_weigh_sm100.cu).
#pragma once

#include "kv8.h"

namespace gtb {
namespace kv8 {

// More rows per (sequence, kv head) than this take the path, for 16-bit q and head sizes up to 128
constexpr int CHUNK_ROWS = 64;
bool chunk_supported(const Kv8AttnArgs& a);
int launch_chunk(const Kv8AttnArgs& a, float* lse, int n_sm, cudaStream_t st);

// score_out from the rows' log-sum-exp (kv8_weigh_sm100.cu)
int launch_weigh(const Kv8AttnArgs& a, const float* lse, cudaStream_t st);

}  // namespace kv8
}  // namespace gtb
