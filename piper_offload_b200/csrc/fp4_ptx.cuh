// fp4_ptx.cuh - the block-scaled tensor-core instructions and the cluster
// helpers that the FP4 products use beside ptx.cuh.
#pragma once
#include <cuda_bf16.h>

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

// 16 lanes x 32 fp32 columns as the fragments of m16n8 matrices, asynchronously:
// registers 4j .. 4j+3 hold row lane / 4 of columns 8j + 2 (lane % 4) and the
// next, then the same of row lane / 4 + 8.
__device__ __forceinline__ void tmem_ld_fragments(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// The registers of two loads, named so that no use moves ahead of the wait.
__device__ __forceinline__ void tmem_ld_fragments_wait(uint32_t (&a)[16], uint32_t (&b)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]), "+r"(a[8]),
                 "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15])
               :
               : "memory");
  asm volatile(""
               : "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]), "+r"(b[5]), "+r"(b[6]), "+r"(b[7]), "+r"(b[8]),
                 "+r"(b[9]), "+r"(b[10]), "+r"(b[11]), "+r"(b[12]), "+r"(b[13]), "+r"(b[14]), "+r"(b[15])
               :
               : "memory");
}

// Four 8x8 matrices of 16-bit values, transposed: lane 8i + r gives the
// address of the 16 bytes that hold column r of matrix i.
__device__ __forceinline__ void stmatrix_trans(uint32_t saddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(saddr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

__device__ __forceinline__ uint32_t bf16_pair(uint32_t lo, uint32_t hi, float alpha) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(lo) * alpha, __uint_as_float(hi) * alpha);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// True in one lane of a converged warp. Tensor-core instructions take their
// operands from uniform registers: under this predicate the compiler keeps
// them there, while under `lane == 0` every one of them costs about 120 cycles.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
  return p != 0u;
}

// A place in a ring of N barriers and the parity of its current round, kept by
// addition: the remainder and quotient of a running count cost more than the
// wait they are for.
template <int N>
struct Ring {
  int slot = 0;
  uint32_t round = 0;  // parity
  __device__ __forceinline__ void next() {
    if (++slot == N) {
      slot = 0;
      round ^= 1u;
    }
  }
  // The place of running count `it`.
  __device__ __forceinline__ void at(int it) {
    slot = it % N;
    round = (it / N) & 1;
  }
};

// ---------------------------------------------------------------- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Every thread of every block of the cluster; what was written before is seen after.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The four fp32 values at this block's shared-memory address `saddr` in block `rank`.
__device__ __forceinline__ float4 load_cluster(uint32_t saddr, uint32_t rank) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

// Programmatic launches: let the next kernel start its own set-up / wait for
// everything the previous one wrote.
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace fp4
