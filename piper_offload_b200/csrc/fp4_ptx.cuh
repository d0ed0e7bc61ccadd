// fp4_ptx.cuh - the block-scaled tensor-core instructions and the cluster
// helpers that the FP4 products use beside ptx.cuh.
#pragma once
#include "ptx.cuh"

namespace fp4 {

// Instruction descriptor of kind::mxf4 / kind::mxf4nvf4, fp32 accumulation,
// e2m1 operands, both K-major, M = 128: bits 4-5 / 29-30 pick the scale byte
// of B / A inside its 32-bit column, bits 7-9 and 10-12 the operand types,
// bits 17-22 N / 8, bit 23 the scale type (1 = ue8m0), bits 24-28 M / 16.
__device__ __forceinline__ constexpr uint32_t idesc_fp4(uint32_t m, uint32_t n, bool e8m0, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((e8m0 ? 1u : 0u) << 23) | ((m >> 4) << 24) |
         (sf_id << 29);
}

// D += A * B over K = 64 with one scale per 16 (NVFP4, four scale bytes of a
// column) or per 32 values (MXFP4, two bytes). The scales' tensor-memory
// addresses are multiples of four columns.
template <int FMT>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  if constexpr (FMT == 1) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  }
}

// One 512-byte scale tile (128 rows x 4 scales) from shared memory to four
// tensor-memory columns: lane r % 32 of column r / 32, in all four lane quarters.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

// Programmatic launches: let the next kernel start its own set-up / wait for
// everything the previous one wrote.
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace fp4
