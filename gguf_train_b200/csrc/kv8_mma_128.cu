// kv8_mma.cuh for head sizes stored as 128 bytes a row.
#include "kv8_mma.cuh"

namespace gtb {
namespace kv8 {

int launch_mma_128(const MmaP& p, int n_sm, cudaStream_t st) {
    return p.c.format == GTB_KV8_INT8 ? launch_mma_rows<128, GTB_KV8_INT8>(p, n_sm, st)
                                      : launch_mma_rows<128, GTB_KV8_E4M3>(p, n_sm, st);
}

}  // namespace kv8
}  // namespace gtb
