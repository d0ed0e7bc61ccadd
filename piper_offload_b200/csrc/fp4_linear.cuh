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
  int32_t items;           // bound on the tiles
  int32_t early;           // the weight is used where it is: loads of it need not wait for the launch before
  int32_t vec;             // rows of y start on 16-byte boundaries
};

template <int FMT, int BN>
struct LinearShape {
  static constexpr int kTiles = FMT == kNV ? 4 : 2;                 // scale tiles per stage and 128 rows
  static constexpr int kXBlocks = (BN + 127) / 128;                 // 128-token scale blocks per tile
  static constexpr int kW = kTileRows * kStageBytes;
  static constexpr int kX = BN * kStageBytes;
  static constexpr int kSW = kTiles * 512;
  static constexpr int kSX = kXBlocks * kTiles * 512;
  static constexpr int kStage = kW + kX + kSW + kSX;
  static constexpr int kOut = 4 * 2048;                             // 32 tokens x 32 outputs of each epilogue warp
  static constexpr int kStages = (kSmemMax - 2048 - kOut) / kStage < 9 ? (kSmemMax - 2048 - kOut) / kStage : 9;
  static constexpr int kSmem = kStages * kStage + kOut + 1024 + 512;
  // tensor memory: two accumulators, then two buffers of scales
  static constexpr int kScaleCols = kTiles * 4 * (1 + kXBlocks);
  static constexpr int kCols = 2 * BN + 2 * kScaleCols;
  static constexpr int kAlloc = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kCols <= 512 && kStages >= 4, "the tile does not fit");
};

// One persistent block per SM. Roles run through the same tiles on their own:
// the producer and the tensor-core warp are up to two accumulators ahead of
// the epilogue.
template <int DT, int FMT, int BN>
__global__ void __launch_bounds__(kLinearThreads, 1) linear_kernel(const __grid_constant__ LinearArgs p) {
  using S = LinearShape<FMT, BN>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  uint8_t* out = smem + S::kStages * S::kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(out + S::kOut);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == 0 && lane == 0) {
    pm::prefetch_tmap(&p.w_map);
    pm::prefetch_tmap(&p.x_map);
    for (int s = 0; s < S::kStages; ++s) {
      pm::mbar_init(&full[s], 1);
      pm::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      pm::mbar_init(&acc_full[b], 1);
      pm::mbar_init(&acc_empty[b], 4);
    }
    pm::fence_mbar_init();
  } else if (warp == 1) {
    pm::tmem_alloc(tmem_at, S::kAlloc);
    pm::tmem_relinquish();
  }
  pm::tc_fence_before();
  __syncthreads();
  pm::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_at, 0);
  const int stages = (p.k_steps + 3) / 4;

  if (warp == 0) {
    Ring<S::kStages> ring;
    int it = 0;  // stages issued
    bool ok = true, waited = false;
    TileAt t;
    for (int id = blockIdx.x; ok && id < p.items && find_tile(p.groups, id, BN, t); id += gridDim.x) {
      if (t.expert == p.groups.experts) continue;
      const int w_row = __shfl_sync(0xFFFFFFFFu, t.expert * p.rows + t.row_tile * kTileRows, 0);
      const int x_row = __shfl_sync(0xFFFFFFFFu, t.first, 0);
      const uint8_t* w_scale =
          p.w_scale + static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, t.expert * p.groups.row_tiles + t.row_tile, 0)) * p.scale_tiles * 512;
      const uint8_t* x_scale = p.x_scale + static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, t.scale_row >> 7, 0)) * p.scale_tiles * 512;
      const auto load_w = [&](int i, int s) {
        uint8_t* at = smem + s * S::kStage;
        const int tiles = min(S::kTiles, p.scale_tiles - i * S::kTiles);
        pm::mbar_arrive_expect_tx(&full[s], S::kW + S::kX + tiles * 512 * (1 + S::kXBlocks));
        pm::tma_load_2d(at, &p.w_map, i * kStageBytes, w_row, &full[s]);
        pm::bulk_g2s(at + S::kW + S::kX, w_scale + static_cast<int64_t>(i) * S::kTiles * 512, tiles * 512, &full[s]);
      };
      const auto load_x = [&](int i, int s) {
        uint8_t* at = smem + s * S::kStage;
        const int tiles = min(S::kTiles, p.scale_tiles - i * S::kTiles);
        pm::tma_load_2d(at + S::kW, &p.x_map, i * kStageBytes, x_row, &full[s]);
#pragma unroll
        for (int b = 0; b < S::kXBlocks; ++b)
          pm::bulk_g2s(at + S::kW + S::kX + S::kSW + b * S::kTiles * 512,
                       x_scale + (static_cast<int64_t>(b) * p.scale_tiles + i * S::kTiles) * 512, tiles * 512, &full[s]);
      };
      if (elect_one()) {
        int i = 0;
        if (!waited) {
          // the first tile: the weight's part of every stage goes out before the tokens are quantized
          const int ahead = p.early ? min(stages, S::kStages) : 0;
          for (int j = 0; j < ahead; ++j) load_w(j, j);
          grid_wait();
          for (; i < ahead; ++i, ++it, ring.next()) load_x(i, i);
        }
        for (; i < stages; ++i, ++it, ring.next()) {
          ok = it < S::kStages || pm::mbar_wait(&empty[ring.slot], ring.round ^ 1u, pm::kStatusTimeoutLoad);
          if (!ok) break;
          load_w(i, ring.slot);
          load_x(i, ring.slot);
        }
      }
      __syncwarp();
      waited = true;
      // the elected lane may be another one next time
      ok = __all_sync(0xFFFFFFFFu, ok);
      it = __reduce_max_sync(0xFFFFFFFFu, it);
      ring.slot = it % S::kStages;
      ring.round = (it / S::kStages) & 1;
    }
    if (!waited) grid_wait();  // no block ends before the launch it depends on
    // the last copies land before the block's shared memory goes, even if the tensor-core warp gave up
    for (int i = max(0, it - S::kStages); i < it; ++i)
      pm::mbar_wait(&full[i % S::kStages], (i / S::kStages) & 1, pm::kStatusTimeoutLoad);
    __syncwarp();
  } else if (warp == 1) {
    Ring<S::kStages> ring, old;  // this stage; the one two stages ago
    int it = 0, n = 0;           // stages used, tiles begun
    bool ok = true;
    TileAt t;
    for (int id = blockIdx.x; ok && id < p.items && find_tile(p.groups, id, BN, t); id += gridDim.x) {
      if (t.expert == p.groups.experts) continue;
      const int b = n & 1;
      const uint32_t d = tmem + b * BN;
      const uint32_t n_mma = (static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, t.count, 0)) + 15u) & ~15u;  // computed token columns
      const uint32_t idesc = idesc_fp4(kTileRows, n_mma, FMT == kMX, 0);
      if (elect_one()) {
        ok = n < 2 || pm::mbar_wait(&acc_empty[b], ((n >> 1) - 1) & 1, pm::kStatusTimeoutMma);
        pm::tc_fence_after();
        for (int i = 0; ok && i < stages; ++i, ++it, ring.next()) {
          // the scale buffer's last readers, two stages ago, have finished
          if (it >= 2) {
            ok = pm::mbar_wait(&empty[old.slot], old.round, pm::kStatusTimeoutMma);
            old.next();
          }
          ok = ok && pm::mbar_wait(&full[ring.slot], ring.round, pm::kStatusTimeoutMma);
          if (!ok) break;
          pm::tc_fence_after();
          const uint32_t at = pm::smem_u32(smem) + ring.slot * S::kStage;
          const uint32_t sw = tmem + 2 * BN + (it & 1) * S::kScaleCols, sx = sw + S::kTiles * 4;
          const int tiles = p.scale_tiles - i * S::kTiles, steps = p.k_steps - i * 4;
          const uint64_t ws = pm::smem_desc(at + S::kW + S::kX, 0, 128);
          const uint64_t xs = pm::smem_desc(at + S::kW + S::kX + S::kSW, 0, 128);
#pragma unroll
          for (int j = 0; j < S::kTiles; ++j) {
            if (j < tiles) {
              tmem_cp_scales(sw + j * 4, ws + j * (512 >> 4));
#pragma unroll
              for (int k = 0; k < S::kXBlocks; ++k)
                tmem_cp_scales(sx + (j * S::kXBlocks + k) * 4, xs + (k * S::kTiles + j) * (512 >> 4));
            }
          }
          const uint64_t a = pm::smem_desc_sw(at, 16, 1024, 2), x = pm::smem_desc_sw(at + S::kW, 16, 1024, 2);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            constexpr uint32_t kSecondHalf = (2u << 4) | (2u << 29);  // scale bytes 2 and 3 of a column
            const uint32_t tile = FMT == kNV ? j : j >> 1;
            if (j < steps)
              umma_fp4<FMT>(d, a + j * 2, x + j * 2, FMT == kMX && (j & 1) ? idesc | kSecondHalf : idesc, sw + tile * 4,
                            sx + tile * 4 * S::kXBlocks, (i | j) != 0);
          }
          pm::umma_commit(&empty[ring.slot]);
        }
        pm::umma_commit(&acc_full[b]);
      }
      __syncwarp();
      ++n;
      // the elected lane may be another one next time
      ok = __all_sync(0xFFFFFFFFu, ok);
      it = __reduce_max_sync(0xFFFFFFFFu, it);
      ring.slot = it % S::kStages;
      ring.round = (it / S::kStages) & 1;
      const int before = max(it - 2, 0);
      old.slot = before % S::kStages;
      old.round = (before / S::kStages) & 1;
    }
    __syncwarp();
  } else {
    const float x_second = p.x_second != nullptr ? *p.x_second : 1.0f;
    uint8_t* mine = out + (warp & 3) * 2048;
    int n = 0;
    TileAt t;
    for (int id = blockIdx.x; id < p.items && find_tile(p.groups, id, BN, t); id += gridDim.x) {
      if (t.expert == p.groups.experts) {
        store_zeros<DT>(p.y, t, p.rows, threadIdx.x - 64, 128);
        continue;
      }
      const int b = n & 1;
      const float alpha = (p.w_second != nullptr ? p.w_second[t.expert] : 1.0f) * x_second;
      const bool ok = pm::mbar_wait(&acc_full[b], (n >> 1) & 1, pm::kStatusTimeoutMma);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      pm::tc_fence_after();
      store_tile<DT>(tmem + b * BN, p.y, t, p.rows, alpha, 0, BN, mine, p.vec != 0);
      pm::tc_fence_before();
      __syncwarp();
      if (lane == 0) pm::mbar_arrive(&acc_empty[b]);
      ++n;
    }
  }
  __syncthreads();
  if (warp == 1) {
    pm::tc_fence_after();
    pm::tmem_dealloc(tmem, S::kAlloc);
  }
}

}  // namespace fp4
