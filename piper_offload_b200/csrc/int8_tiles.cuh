// int8_tiles.cuh - from a finished tile in tensor memory to rows of the result, for the INT8 products and gradients.
#pragma once
#include "fp4_tiles.cuh"
#include "int8_quant.cuh"

namespace i8 {

using fp4::kSmemMax;
using fp4::kTileRows;
using fp4::TileAt;

// Columns of tensor memory are allocated in powers of two from 32 on (any other number is an illegal instruction).
__host__ __device__ constexpr int tmem_columns(int used) { return used <= 32 ? 32 : used <= 64 ? 64 : used <= 128 ? 128 : used <= 256 ? 256 : 512; }

// kind::i8: signed 8-bit operands, both K-major, 32-bit sums, M = 128.
__host__ __device__ constexpr uint32_t idesc_i8(uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// kind::f16: fp16 operands, fp32 sums, A stored M-major (bit 15), B K-major.
__host__ __device__ constexpr uint32_t idesc_grad(uint32_t n, uint32_t m) { return (1u << 4) | (1u << 15) | ((n >> 3) << 17) | ((m >> 4) << 24); }

// ------------------------------------------------------------ pairs of SMs (cta_group::2)
// Arrive once on the barrier at this place in both blocks when every product issued before is done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(pm::smem_u32(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}

// A tile into this block's shared memory, counted on the barrier at `bar` of the cluster's address space: the even block's.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* tmap, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(pm::smem_u32(dst)),
      "l"(tmap), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// The cluster's address of this block's shared-memory address in block `rank`.
__device__ __forceinline__ uint32_t in_block(uint32_t saddr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(saddr), "r"(rank));
  return remote;
}

// One arrival on the barrier at `bar` of the cluster's address space. What the thread has written, or has seen through barriers
// of its block, is there for a thread of either block that waits with mbar_wait_pair; with the default scope it would be
// for threads of the arriving block alone. The thread waits for all that it has under way: a warp with loads in flight
// arrives in its own block, where another passes it on (the gradient's decoding warps themselves took 318 us so, 2048 x
// 14336 x 4096).
__device__ __forceinline__ void mbar_arrive_pair(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// The threads of a pair wait for everything that the other block may have a part in with the scope of the cluster too.
__device__ __forceinline__ bool mbar_try_wait_pair(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(pm::smem_u32(bar)), "r"(parity), "r"(pm::kSuspendHintNs)
      : "memory");
  return ok != 0;
}

// pm::mbar_wait of such a thread.
__device__ __forceinline__ bool mbar_wait_pair(uint64_t* bar, uint32_t parity, unsigned int code) {
  if (mbar_try_wait_pair(bar, parity)) return true;
  const uint64_t t0 = pm::global_timer_ns();
  for (uint32_t spin = 0;; ++spin) {
    if (mbar_try_wait_pair(bar, parity)) return true;
    if ((spin & 63u) == 63u && pm::global_timer_ns() - t0 > pm::kWaitLimitNs) {
      atomicOr(&pm::g_status, code);
      return false;
    }
  }
}

template <bool kPair>
__device__ __forceinline__ bool mbar_wait_of(uint64_t* bar, uint32_t parity, unsigned int code) {
  if constexpr (kPair) return mbar_wait_pair(bar, parity, code);
  else return pm::mbar_wait(bar, parity, code);
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pm::smem_u32(dst)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}

template <int DT>
__device__ __forceinline__ void store_value(void* y, int64_t at, float v) {
  if constexpr (DT == kBF16) static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else if constexpr (DT == kF16) static_cast<__half*>(y)[at] = __float2half_rn(v);
  else static_cast<float*>(y)[at] = v;
}

template <int DT>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
  if constexpr (DT == kBF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

template <int DT>
__device__ __forceinline__ void zero_tile(void* y, const TileAt& t, int cols, int thread, int threads) {
  const int c0 = t.row_tile * kTileRows, n = min(kTileRows, cols - c0);
  for (int i = thread; i < t.count * kTileRows; i += threads)
    if ((i & (kTileRows - 1)) < n)
      store_value<DT>(y, static_cast<int64_t>(t.first + i / kTileRows) * cols + c0 + (i & (kTileRows - 1)), 0.0f);
}

// What a sum of a product becomes: (sum - zero point * the token's sum of codes) * the token's scale * the row's scale,
// the difference exact in 32 bits. Of a gradient: the sum times the token's power of two.
template <bool kInt>
struct Outcome {
  float row_scale;
  int32_t zero;
  __device__ __forceinline__ float of(uint32_t sum, float token_scale, int32_t token_sum) const {
    if constexpr (kInt) return static_cast<float>(static_cast<int32_t>(sum) - zero * token_sum) * token_scale * row_scale;
    else return __uint_as_float(sum) * token_scale;
  }
};

// The scales and zero points of the weight's rows.
struct RowsOf {
  RowScales scales;
  const int8_t* zero;  // or NULL
  int32_t zero_step;

  template <bool kInt>
  __device__ __forceinline__ Outcome<kInt> outcome(int64_t row, bool exists) const {
    Outcome<kInt> o{0.0f, 0};
    if (kInt && exists) {
      o.row_scale = row_scale(scales, row);
      if (zero != nullptr) o.zero = zero[row * zero_step];
    }
    return o;
  }
};

// Four epilogue warps' share of a finished tile: tensor-memory lane = column of y, tensor-memory column = token. 16-bit
// results leave as in the FP4 products: fragments of 8x8 matrices, transposed by stmatrix into the warp's own 2 KB of shared
// memory (`stage`) and out in 16-byte pieces of y's rows; fp32 in runs of 128 bytes. `scale` and `sums` are the tile's
// tokens' in shared memory. `row0`: the weight's row of the tile's expert that is column 0 of y.
template <int DT, bool kInt>
__device__ __forceinline__ void store_tile(uint32_t tmem, void* y, const TileAt& t, int cols, const RowsOf& rows, int64_t row0,
                                           const float* scale, const int32_t* sums, int from_col, int to_col, uint8_t* stage, bool vec) {
  const int quarter = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const int n0 = t.row_tile * kTileRows + quarter * 32;
  const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const int end = min(to_col, t.count);
  if constexpr (DT != kF32) {
    Outcome<kInt> o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = n0 + (lane >> 2) + 8 * k;
      o[k] = rows.template outcome<kInt>(row0 + n, n < cols);
    }
    const uint32_t base = pm::smem_u32(stage);
    const int piece = lane & 3;
    const int left = cols - n0 - piece * 8;  // outputs of this lane's piece that exist
    for (int c = from_col; c < end; c += 32) {
      uint32_t lo[16], hi[16];
      fp4::tmem_ld_fragments(at + c, lo);
      fp4::tmem_ld_fragments(at + (16u << 16) + c, hi);
      fp4::tmem_ld_fragments_wait(lo, hi);
      __syncwarp();  // the warp has read the last 32 tokens out of its stage
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int pair = c + 8 * j + 2 * piece;
        const float2 s = *reinterpret_cast<const float2*>(scale + pair);
        int2 q = make_int2(0, 0);
        if (kInt) q = *reinterpret_cast<const int2*>(sums + pair);
        const int token = j * 8 + (lane & 7);
        const uint32_t to = base + token * 64 + (((lane >> 3) ^ ((token >> 1) & 3)) << 4);
        const auto both = [&](const uint32_t (&r)[16], int k, int half) {
          return pair16<DT>(o[k].of(r[4 * j + half], s.x, q.x), o[k].of(r[4 * j + half + 1], s.y, q.y));
        };
        fp4::stmatrix_trans(to, both(lo, 0, 0), both(lo, 1, 2), both(hi, 2, 0), both(hi, 3, 2));
      }
      __syncwarp();
      uint16_t* row = static_cast<uint16_t*>(y) + (static_cast<int64_t>(t.first + c + (lane >> 2)) * cols + n0 + piece * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j, row += static_cast<int64_t>(8) * cols) {
        const int token = j * 8 + (lane >> 2);
        const uint4 v = *reinterpret_cast<const uint4*>(stage + token * 64 + ((piece ^ ((token >> 1) & 3)) << 4));
        if (c + token >= end) break;
        if (vec && left >= 8) {
          *reinterpret_cast<uint4*>(row) = v;
        } else {
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < left) row[k] = static_cast<uint16_t>(w[k >> 1] >> (16 * (k & 1)));
        }
      }
    }
  } else {
    const int n = n0 + lane;
    const Outcome<kInt> o = rows.template outcome<kInt>(row0 + n, n < cols);
    for (int c = from_col; c < end; c += 32) {
      float v[32];
      pm::tmem_ld32(at + c, v);
      if (n < cols) {
        float* to = static_cast<float*>(y) + (static_cast<int64_t>(t.first + c) * cols + n);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < end) to[static_cast<int64_t>(j) * cols] = o.of(__float_as_uint(v[j]), scale[c + j], kInt ? sums[c + j] : 0);
      }
    }
  }
}

// A block adds up its share of a tile over the cluster, in rank order, and stores it: four outputs of a token a thread, the
// ranks' values all in flight at once. Sums of a product are whole numbers, so their order changes nothing.
template <int DT, bool kInt>
__device__ __forceinline__ void add_cluster_sums(const float* parts, void* y, const TileAt& t, int cols, const RowsOf& rows, int64_t row0,
                                                 const float* scale, const int32_t* sums, int rank, int split, int threads, bool vec) {
  const uint32_t base = pm::smem_u32(parts);
  const int n0 = t.row_tile * kTileRows;
  for (int i = rank * threads + threadIdx.x; i < t.count * (kTileRows / 4); i += split * threads) {
    const int n = n0 + (i % (kTileRows / 4)) * 4, token = i / (kTileRows / 4);
    if (n >= cols) continue;
    float4 v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < split) v[r] = fp4::load_cluster(base + i * 16, r);
    uint32_t sum[4] = {__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[0].z), __float_as_uint(v[0].w)};
#pragma unroll
    for (int r = 1; r < 8; ++r)
      if (r < split) {
        const float add[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          sum[k] = kInt ? sum[k] + __float_as_uint(add[k]) : __float_as_uint(__uint_as_float(sum[k]) + add[k]);
      }
    float f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      f[k] = rows.template outcome<kInt>(row0 + n + k, n + k < cols).of(sum[k], scale[token], kInt ? sums[token] : 0);
    const int64_t at = static_cast<int64_t>(t.first + token) * cols + n;
    if (vec) {  // rows are 16-byte aligned, so the four outputs exist and lie together
      if constexpr (DT != kF32) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(y) + at) = make_uint2(pair16<DT>(f[0], f[1]), pair16<DT>(f[2], f[3]));
      else *reinterpret_cast<float4*>(static_cast<float*>(y) + at) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < cols) store_value<DT>(y, at + k, f[k]);
    }
  }
}

}  // namespace i8
