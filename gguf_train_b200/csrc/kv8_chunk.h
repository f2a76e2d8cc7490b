// The tcgen05 paths of kv8_attention for many query rows (kv8_chunk_sm100.cu, kv8_weigh_sm100.cu).
#pragma once

#include "kv8.h"

namespace gtb {
namespace kv8 {

// More rows per (sequence, kv head) than this take the path, for 16-bit q and head sizes up to 128: making the cache f16
// costs more than few rows gain. kv8_mma.cuh / this path, us, 32 sequences of 100 to 8k tokens, 8 kv heads of 128:
// 32 rows 150 / 339, 64 254 / 345, 68 386 / 338, 128 516 / 341, 512 1960 / 453. 68 and 128 rows at full caches of 512, 2048 and
// 8192 tokens: one sequence 25, 41, 66 / 27, 27, 46 and 25, 41, 56 / 21, 28, 47; 32 sequences 89, 179, 529 / 56, 177, 582 and
// 109, 232, 704 / 58, 179, 585. One sequence of 128 tokens is a few launches either way (19 / 19 to 27).
constexpr int CHUNK_ROWS = 64;
bool chunk_supported(const Kv8AttnArgs& a);
int launch_chunk(const Kv8AttnArgs& a, float* lse, int n_sm, cudaStream_t st);

// score_out from the rows' log-sum-exp (kv8_weigh_sm100.cu)
int launch_weigh(const Kv8AttnArgs& a, const float* lse, cudaStream_t st);

}  // namespace kv8
}  // namespace gtb
