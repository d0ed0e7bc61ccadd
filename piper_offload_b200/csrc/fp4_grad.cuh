// fp4_grad.cuh - dx[t, k] = alpha * sum_n dy[t, n] * w[n, k] with w in packed FP4.
//
// The sum runs over the weight's rows while its scales run along them, so the
// block-scaled instructions do not apply. Instead the weight is decoded on
// chip to bf16, which holds every code times its block scale exactly (at most
// 2 + 4 significant bits), and multiplied on the bf16 tensor pipe with fp32
// sums. A tile is 128 columns of w (the 128-row operand, stored with its
// columns contiguous) x up to BN tokens; a stage is 64 rows of w. dy comes by
// bulk tensor copies; eight warps decode: 16 bytes of codes a thread and
// stage, loaded two stages ahead, looked up by byte permutes, scaled by packed
// bf16 products and written in the 128-byte swizzle.
//
// fp32 gradients are the sum of three bf16 terms (24 bits): the stages go
// over the weight once per term.
#pragma once
#include <cuda.h>

#include "fp4_ptx.cuh"
#include "fp4_tiles.cuh"

namespace fp4 {

constexpr int kGradStageRows = 64;   // rows of w per stage
constexpr int kGradThreads = 320;    // producer warp, tensor-core warp, eight decoding and epilogue warps
constexpr int kDecodeWarps = 8;

struct GradArgs {
  CUtensorMap dy_map;   // (terms * tokens, rows of w) bf16
  const uint8_t* codes;
  const uint8_t* scale;
  const float* second;  // (experts) or NULL
  Groups groups;        // row tiles: of 128 columns of w
  void* dx;
  int64_t code_pitch;
  int32_t rows, cols;   // of w
  int32_t swizzled;
  int32_t scale_cols;   // scales, or tiles of them, per row
  int32_t terms;
  int32_t vec;          // rows of dx start on 16-byte boundaries
  int32_t piece;        // bytes that aligned loads of codes may take: 16, 8 or 1
};

template <int BN>
struct GradShape {
  static constexpr int kA = kGradStageRows * kTileRows * 2;
  static constexpr int kB = BN * kGradStageRows * 2;
  static constexpr int kStage = kA + kB;
  static constexpr int kCtas = BN <= 128 ? 2 : 1;
  static constexpr int kStages = (kSmemMax / kCtas - 3072) / kStage < 5 ? (kSmemMax / kCtas - 3072) / kStage : 5;
  static constexpr int kSmem = kStages * kStage + 1024 + 256;
  static constexpr int kAlloc = BN < 32 ? 32 : BN;
};

// kind::f16, bf16 operands, fp32 sums, A stored M-major (bit 15), B K-major, M = 128.
__device__ __forceinline__ constexpr uint32_t idesc_grad(uint32_t n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// A thread's share of a stage: 32 codes of one row and their scales as bf16 pairs.
struct Piece {
  uint4 codes;
  uint32_t scale[2];  // MXFP4: both the same
};

template <int FMT>
__device__ __forceinline__ Piece load_piece(const GradArgs& p, int64_t expert, int row, int col) {
  Piece out;
  out.codes = make_uint4(0u, 0u, 0u, 0u);
  out.scale[0] = out.scale[1] = 0u;
  if (row >= p.rows || col >= p.cols) return out;
  const int64_t r = expert * p.rows + row;
  const uint8_t* c = p.codes + r * p.code_pitch + (col >> 1);
  const int bytes = min(16, (p.cols - col) >> 1);  // 16, or 8 at the end of a row
  if (p.piece == 16 && bytes == 16) {
    out.codes = *reinterpret_cast<const uint4*>(c);
  } else if (p.piece >= 8) {
    const uint2 lo = *reinterpret_cast<const uint2*>(c);
    out.codes.x = lo.x;
    out.codes.y = lo.y;
    if (bytes == 16) {
      const uint2 hi = *reinterpret_cast<const uint2*>(c + 8);
      out.codes.z = hi.x;
      out.codes.w = hi.y;
    }
  } else {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < bytes) w[i >> 2] |= static_cast<uint32_t>(c[i]) << (8 * (i & 3));
    out.codes = make_uint4(w[0], w[1], w[2], w[3]);
  }
  const int block = col / block_values<FMT>();
  const int64_t tiles = (static_cast<int64_t>(p.rows) + 127) >> 7;
  const uint8_t* s = p.swizzled ? p.scale + expert * tiles * p.scale_cols * 512 + swizzled_byte(row, block, p.scale_cols)
                                : p.scale + r * p.scale_cols + block;
  out.scale[0] = out.scale[1] = s[0];
  if (FMT == kNV && bytes == 16) out.scale[1] = s[1];  // an even block and the next are in one tile
  return out;
}

template <int DT, int FMT, int BN>
__global__ void __launch_bounds__(kGradThreads, GradShape<BN>::kCtas) grad_kernel(const __grid_constant__ GradArgs p) {
  using S = GradShape<BN>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kStages * S::kStage);  // dy landed
  uint64_t* ready = full + S::kStages;                                          // w decoded
  uint64_t* empty = ready + S::kStages;
  uint64_t* done = empty + S::kStages;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);
  int32_t* have = reinterpret_cast<int32_t*>(tmem_at + 1);
  TileAt* shared_tile = reinterpret_cast<TileAt*>(have + 1);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == 0) {
    TileAt t;
    const bool ok = find_tile(p.groups, blockIdx.x, BN, t);
    if (lane == 0) {
      *have = ok;
      if (ok) *shared_tile = t;
      pm::prefetch_tmap(&p.dy_map);
      for (int s = 0; s < S::kStages; ++s) {
        pm::mbar_init(&full[s], 1);
        pm::mbar_init(&ready[s], kDecodeWarps);
        pm::mbar_init(&empty[s], 1);
      }
      pm::mbar_init(done, 1);
      pm::fence_mbar_init();
    }
  } else if (warp == 1) {
    pm::tmem_alloc(tmem_at, S::kAlloc);
    pm::tmem_relinquish();
  }
  pm::tc_fence_before();
  __syncthreads();
  pm::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_at, 0);
  const TileAt t = *shared_tile;
  const int blocks = (p.rows + kGradStageRows - 1) / kGradStageRows;  // of 64 rows of w
  const int stages = blocks * p.terms;
  const uint32_t n_mma = static_cast<uint32_t>((t.count + 15) & ~15);

  if (*have && t.expert == p.groups.experts) {
    store_zeros<DT>(p.dx, t, p.cols, threadIdx.x, kGradThreads);
  } else if (*have) {
    if (warp == 0) {
      grid_wait();
      const int first = __shfl_sync(0xFFFFFFFFu, t.first, 0);
      int issued = 0, block = 0, row = first;
      for (int i = 0; i < stages; ++i) {
        const int s = i % S::kStages;
        const bool ok = i < S::kStages || pm::mbar_wait(&empty[s], ((i / S::kStages) - 1) & 1, pm::kStatusTimeoutLoad);
        if (!__all_sync(0xFFFFFFFFu, ok)) break;
        if (elect_one()) {
          pm::mbar_arrive_expect_tx(&full[s], S::kB);
          pm::tma_load_2d(smem + s * S::kStage + S::kA, &p.dy_map, block * kGradStageRows, row, &full[s]);
        }
        __syncwarp();
        issued = i + 1;
        if (++block == blocks) {  // the next term
          block = 0;
          row += static_cast<int>(p.groups.tokens);
        }
      }
      // the last copies land before the block's shared memory goes, even if the tensor-core warp gave up
      for (int i = max(0, issued - S::kStages); i < issued; ++i)
        pm::mbar_wait(&full[i % S::kStages], (i / S::kStages) & 1, pm::kStatusTimeoutLoad);
      __syncwarp();
    } else if (warp == 1) {
      const uint32_t idesc = idesc_grad(__shfl_sync(0xFFFFFFFFu, n_mma, 0));
      for (int i = 0; i < stages; ++i) {
        const int s = i % S::kStages;
        const bool ok = pm::mbar_wait(&full[s], (i / S::kStages) & 1, pm::kStatusTimeoutMma) &&
                        pm::mbar_wait(&ready[s], (i / S::kStages) & 1, pm::kStatusTimeoutMma);
        if (!__all_sync(0xFFFFFFFFu, ok)) break;
        pm::tc_fence_after();
        const uint32_t at = pm::smem_u32(smem) + s * S::kStage;
        if (elect_one()) {
          // w: 64-column blocks 8 KB apart, groups of 8 rows 1 KB apart; dy: 128-byte rows of 64 values
          const uint64_t a = pm::smem_desc_sw(at, kGradStageRows * 128, 1024, 2);
          const uint64_t b = pm::smem_desc_sw(at + S::kA, 16, 1024, 2);
#pragma unroll
          for (int j = 0; j < kGradStageRows / 16; ++j)
            pm::umma_f16(tmem, a + j * (2048 >> 4), b + j * (32 >> 4), idesc, (i | j) != 0);
          pm::umma_commit(&empty[s]);
          if (i + 1 == stages) pm::umma_commit(done);
        }
        __syncwarp();
      }
      __syncwarp();
    } else {
      const int tid = threadIdx.x - 64;
      const int r = tid >> 2, quarter = tid & 3;  // row of the stage, 32 columns of the tile
      const int col = t.row_tile * kTileRows + quarter * 32;
      Piece ahead[2];
      ahead[0] = load_piece<FMT>(p, t.expert, r, col);
      ahead[1] = load_piece<FMT>(p, t.expert, (1 % blocks) * kGradStageRows + r, col);
      int next = 2 % blocks;
      bool ok = true;
      for (int i = 0; i < stages && ok; ++i) {
        const int s = i % S::kStages;
        const Piece now = ahead[0];
        ahead[0] = ahead[1];
        if (i + 2 < stages) ahead[1] = load_piece<FMT>(p, t.expert, next * kGradStageRows + r, col);
        if (++next == blocks) next = 0;
        uint32_t w[16];
        const uint32_t c[4] = {now.codes.x, now.codes.y, now.codes.z, now.codes.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const __nv_bfloat162 scale = __float2bfloat162_rn(scale_value<FMT>(now.scale[q >> 1]));
          decode4(c[q], scale, w[4 * q], w[4 * q + 1]);
          decode4(c[q] >> 16, scale, w[4 * q + 2], w[4 * q + 3]);
        }
        if (i >= S::kStages) ok = __all_sync(0xFFFFFFFFu, pm::mbar_wait(&empty[s], ((i / S::kStages) - 1) & 1, pm::kStatusTimeoutLoad));
        if (!ok) break;
        uint8_t* row = smem + s * S::kStage + (quarter >> 1) * (kGradStageRows * 128) + r * 128;
        // the two column blocks go through their 16-byte pieces in another order, so that eight lanes hit eight banks
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int piece = q ^ ((quarter >> 1) * 2);
          uint4 v;
          if (quarter >> 1) v = make_uint4(w[4 * (q ^ 2)], w[4 * (q ^ 2) + 1], w[4 * (q ^ 2) + 2], w[4 * (q ^ 2) + 3]);
          else v = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
          *reinterpret_cast<uint4*>(row + ((((quarter & 1) * 4 + piece) ^ (r & 7)) << 4)) = v;
        }
        pm::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) pm::mbar_arrive(&ready[s]);
      }
      float alpha = 1.0f;
      if (p.second != nullptr) alpha = p.second[t.expert];
      ok = __all_sync(0xFFFFFFFFu, pm::mbar_wait(done, 0, pm::kStatusTimeoutMma));
      pm::tc_fence_after();
      if (ok) {
        // the sums are complete, so the stages are free: each warp takes 2 KB of them
        uint8_t* mine = smem + (warp - 2) * 2048;
        if constexpr (BN >= 64) {  // two warps share each quarter of the lanes: halves of the tokens
          const int half = warp >= 6;
          store_tile<DT>(tmem, p.dx, t, p.cols, alpha, half * (BN / 2), (half + 1) * (BN / 2), mine, p.vec != 0);
        } else if (warp < 6) {
          store_tile<DT>(tmem, p.dx, t, p.cols, alpha, 0, BN, mine, p.vec != 0);
        }
      }
      pm::tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 1) {
    pm::tc_fence_after();
    pm::tmem_dealloc(tmem, S::kAlloc);
  }
}

// dy as rows that bulk copies can read: bf16 as it is, fp32 as three bf16
// terms, each the rounding of what the terms before it left.
template <int DT>
__global__ void __launch_bounds__(256) split_kernel(const void* dy, int64_t stride, int64_t tokens, int32_t rows,
                                                    int64_t pitch, __nv_bfloat16* out) {
  const int64_t per = (rows + 255) / 256;
  const int64_t token = blockIdx.x / per;
  const int n = static_cast<int>(blockIdx.x - token * per) * 256 + threadIdx.x;
  if (n >= rows) return;
  const int64_t at = token * pitch + n;
  if constexpr (DT == kBF16) {
    out[at] = static_cast<const __nv_bfloat16*>(dy)[token * stride + n];
  } else {
    float v = static_cast<const float*>(dy)[token * stride + n];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const __nv_bfloat16 b = __float2bfloat16_rn(v);
      out[i * tokens * pitch + at] = b;
      v = __fsub_rn(v, __bfloat162float(b));
      if (!isfinite(__bfloat162float(b))) v = 0.0f;  // an infinity or a NaN is its first term alone
    }
  }
}

}  // namespace fp4
