// fp4_linear.cuh - y[t, n] = alpha * sum_k x[t, k] * w[n, k] with both operands in packed FP4.
//
// The weight's rows are the tensor core's 128-row operand and the tokens its
// N side, so a tile is 128 outputs x up to BN tokens and the instruction's N
// follows the tokens that are there: experts with few rows waste little.
// A K step is 64 values (32 bytes a row). Operand tiles come by bulk tensor
// copies in the 128-byte swizzle (256 values a row and stage), block scales as
// whole 512-byte tiles of the swizzled layout, from shared memory to tensor
// memory by tcgen05.cp ahead of the products that use them. The scales are
// applied inside the tensor core; sums are fp32 in tensor memory, and the one
// rounding is that of the output.
#pragma once
#include <cuda.h>

#include "fp4_ptx.cuh"
#include "fp4_quant.cuh"
#include "fp4_tiles.cuh"

namespace fp4 {

constexpr int kStageCols = 256;      // K values per stage
constexpr int kStageBytes = kStageCols / 2;
constexpr int kLinearThreads = 192;  // producer warp, tensor-core warp, four epilogue warps

struct LinearArgs {
  CUtensorMap w_map, x_map;
  const uint8_t* w_scale;  // swizzled tiles, experts on 128-row tiles
  const uint8_t* x_scale;  // swizzled tiles, rows as first_scale_row places them
  const float* w_second;   // (experts) or NULL
  const float* x_second;   // one or NULL
  Groups groups;           // row tiles: of 128 outputs
  void* y;
  int32_t rows;            // outputs per expert
  int32_t k_steps;         // of 64 values
  int32_t scale_tiles;     // tiles of 4 scales per row (weight and tokens alike)
};

template <int FMT, int BN>
struct LinearShape {
  static constexpr int kTiles = FMT == kNV ? 4 : 2;                 // scale tiles per stage and 128 rows
  static constexpr int kXBlocks = BN > 128 ? BN / 128 : 1;          // 128-token scale blocks per tile
  static constexpr int kW = kTileRows * kStageBytes;
  static constexpr int kX = BN * kStageBytes;
  static constexpr int kSW = kTiles * 512;
  static constexpr int kSX = kXBlocks * kTiles * 512;
  static constexpr int kStage = kW + kX + kSW + kSX;
  static constexpr int kCtas = BN <= 128 ? 2 : 1;                   // resident per SM
  static constexpr int kStages = (kSmemMax / kCtas - 3072) / kStage < 8 ? (kSmemMax / kCtas - 3072) / kStage : 8;
  static constexpr int kSmem = kStages * kStage + 1024 + 256;
  // tensor memory: accumulator, then two buffers of scales
  static constexpr int kScaleCols = kTiles * 4 * (1 + kXBlocks);
  static constexpr int kCols = BN + 2 * kScaleCols;
  static constexpr int kAlloc = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
};

template <int DT, int FMT, int BN>
__global__ void __launch_bounds__(kLinearThreads, LinearShape<FMT, BN>::kCtas)
    linear_kernel(const __grid_constant__ LinearArgs p) {
  using S = LinearShape<FMT, BN>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kStages * S::kStage);
  uint64_t* empty = full + S::kStages;
  uint64_t* done = empty + S::kStages;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);
  TileAt* shared_tile = reinterpret_cast<TileAt*>(tmem_at + 2);
  int32_t* have = reinterpret_cast<int32_t*>(shared_tile + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    TileAt t;
    const bool ok = find_tile(p.groups, blockIdx.x, BN, t);
    if (lane == 0) {
      *have = ok;
      if (ok) *shared_tile = t;
      pm::prefetch_tmap(&p.w_map);
      pm::prefetch_tmap(&p.x_map);
      for (int s = 0; s < S::kStages; ++s) {
        pm::mbar_init(&full[s], 1);
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
  const uint32_t tmem = *tmem_at;
  const TileAt t = *shared_tile;
  const int stages = (p.k_steps + 3) / 4;
  // token columns that the tensor core computes
  const uint32_t n_mma = static_cast<uint32_t>((t.count + 15) & ~15);

  if (*have && t.expert == p.groups.experts) {
    store_zeros<DT>(p.y, t, p.rows);
  } else if (*have) {
    if (warp == 0) {
      if (lane == 0) {
        const int64_t w_row = static_cast<int64_t>(t.expert) * p.rows + t.row_tile * kTileRows;
        const uint8_t* w_scale =
            p.w_scale + (static_cast<int64_t>(t.expert) * p.groups.row_tiles + t.row_tile) * p.scale_tiles * 512;
        const uint8_t* x_scale = p.x_scale + static_cast<int64_t>(t.scale_row >> 7) * p.scale_tiles * 512;
        grid_wait();
        int issued = 0;
        for (int i = 0; i < stages; ++i) {
          const int s = i % S::kStages;
          if (i >= S::kStages && !pm::mbar_wait(&empty[s], ((i / S::kStages) - 1) & 1, pm::kStatusTimeoutLoad)) break;
          uint8_t* at = smem + s * S::kStage;
          const int tiles = min(S::kTiles, p.scale_tiles - i * S::kTiles);
          pm::mbar_arrive_expect_tx(&full[s], S::kW + S::kX + tiles * 512 * (1 + S::kXBlocks));
          pm::tma_load_2d(at, &p.w_map, i * kStageBytes, static_cast<int>(w_row), &full[s]);
          pm::tma_load_2d(at + S::kW, &p.x_map, i * kStageBytes, t.first, &full[s]);
          pm::bulk_g2s(at + S::kW + S::kX, w_scale + static_cast<int64_t>(i) * S::kTiles * 512, tiles * 512, &full[s]);
#pragma unroll
          for (int b = 0; b < S::kXBlocks; ++b)
            pm::bulk_g2s(at + S::kW + S::kX + S::kSW + b * S::kTiles * 512,
                         x_scale + (static_cast<int64_t>(b) * p.scale_tiles + i * S::kTiles) * 512, tiles * 512, &full[s]);
          issued = i + 1;
        }
        // the last copies land before the block's shared memory goes, even if the tensor-core warp gave up
        for (int i = max(0, issued - S::kStages); i < issued; ++i)
          pm::mbar_wait(&full[i % S::kStages], (i / S::kStages) & 1, pm::kStatusTimeoutLoad);
      }
      __syncwarp();
    } else if (warp == 1) {
      if (lane == 0) {
        for (int i = 0; i < stages; ++i) {
          const int s = i % S::kStages;
          // the scale buffer's last readers, two stages ago, have finished
          if (i >= 2 && !pm::mbar_wait(&empty[(i - 2) % S::kStages], ((i - 2) / S::kStages) & 1, pm::kStatusTimeoutMma)) break;
          if (!pm::mbar_wait(&full[s], (i / S::kStages) & 1, pm::kStatusTimeoutMma)) break;
          pm::tc_fence_after();
          const uint32_t at = pm::smem_u32(smem + s * S::kStage);
          const uint32_t sw = tmem + BN + (i & 1) * S::kScaleCols, sx = sw + S::kTiles * 4;
          const int tiles = min(S::kTiles, p.scale_tiles - i * S::kTiles);
          for (int j = 0; j < tiles; ++j) {
            tmem_cp_scales(sw + j * 4, pm::smem_desc(at + S::kW + S::kX + j * 512, 0, 128));
#pragma unroll
            for (int b = 0; b < S::kXBlocks; ++b)
              tmem_cp_scales(sx + (j * S::kXBlocks + b) * 4,
                             pm::smem_desc(at + S::kW + S::kX + S::kSW + (b * S::kTiles + j) * 512, 0, 128));
          }
          const uint64_t a = pm::smem_desc_sw(at, 16, 1024, 2), b = pm::smem_desc_sw(at + S::kW, 16, 1024, 2);
          const int steps = min(4, p.k_steps - i * 4);
          for (int j = 0; j < steps; ++j) {
            const uint32_t tile = FMT == kNV ? j : j >> 1, id = FMT == kNV ? 0u : (j & 1) * 2u;
            umma_fp4<FMT>(tmem, a + j * 2, b + j * 2, idesc_fp4(kTileRows, n_mma, FMT == kMX, id), sw + tile * 4,
                          sx + tile * 4 * S::kXBlocks, (i | j) != 0);
          }
          pm::umma_commit(&empty[s]);
        }
        pm::umma_commit(done);
      }
      __syncwarp();
    } else {
      float alpha = 1.0f;
      if (p.w_second != nullptr) alpha = p.w_second[t.expert];
      if (p.x_second != nullptr) alpha *= *p.x_second;
      const bool ok = pm::mbar_wait(done, 0, pm::kStatusTimeoutMma);
      pm::tc_fence_after();
      if (__all_sync(0xFFFFFFFFu, ok)) store_tile<DT>(tmem, p.y, t, p.rows, alpha, 0, BN);
      pm::tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 1) {
    pm::tc_fence_after();
    pm::tmem_dealloc(tmem, S::kAlloc);
  }
}

}  // namespace fp4
