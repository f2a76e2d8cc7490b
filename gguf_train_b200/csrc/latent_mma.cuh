// Issue of tcgen05 products by a whole warp on uniform registers, for the latent attention kernels.
//
// One elected lane issues, but the whole warp goes through the loops around it without diverging, on values that are the same in every
// lane for the compiler too (votes and reductions), so that descriptors are formed in uniform registers, where the
// instruction takes its operands from. One lane in loops of its own took 106 cycles a product whatever its size; this way a
// product takes the unit's own time: 33 cycles for M = 64, N = 64, 50 for M = 128, N = 64, 65 for M = 128, N = 128 (K = 16; with both
// operands in shared memory its bandwidth is the bound up to N = 128).
#pragma once

#include "sm100_ptx.cuh"

namespace gtb {
namespace sm100 {

__device__ __forceinline__ bool elect_lane() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ int uniform(int v) { return __reduce_max_sync(~0u, v); }  // of a value that all lanes have

// the same bounded wait taken by a whole warp: every lane gets the same answer
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code));
}

// The low words of operand descriptors (address, leading byte offset) come in registers; the high ones are the same for all
// operands here (stride byte offset 1024, version, 128-byte swizzle).
constexpr uint32_t DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (uint32_t)desc_sw128(saddr, lbo, 1024); }

__device__ __forceinline__ void mma_ss_lo(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void mma_ts_lo(uint32_t d_tmem, uint32_t a_tmem, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI)
        : "memory");
}

// two floats -> one 32-bit word of two 16-bit values (lo in the low half), round to nearest even
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace sm100
}  // namespace gtb
