// int8_linear.cuh - y[t, n] = s_x[t] s_w[n] sum_k q[t, k] (w[n, k] - z[n]) on the 8-bit integer tensor pipe.
//
// The weight's rows are the tensor core's 128-row operand and the tokens its N side, so that the instruction's N follows the
// tokens that are there. A stage is 128 columns: 128-byte rows of both operands by bulk tensor copies in the 128-byte
// swizzle. Sums are whole numbers of 32 bits (at most 65536 columns: 65536 * 127 * 255 < 2^31, so none wraps), the zero
// point's share z[n] sum_k q[t, k] is taken off them exactly, and the roundings are those of the sum to fp32, of the two
// products with the scales, and of the result to its type.
//
// Tokens are quantised by a launch before, which the set-up and the first loads of the weight overlap. Tiles are 32, 64,
// 128 or 256 tokens wide. Where there are too few tiles for the SMs, a cluster of blocks splits K; each leaves its sums in its own
// shared memory and every block adds up its share of the tokens over the cluster.
//
// With few tokens a weight the weight's bytes bound it (16 rows of 8 experts of 14336 x 4096 59 us, 6.0 TB/s for the 353 MB
// of the experts that have rows). With some hundred a weight no unit is near its rate (4096 rows of 32 experts of 2048 x 2048
// 38 us, 8 of them quantising; L2 31 %, DRAM 45 %, tensor pipe 28 %, issue 15 %): waiting for operands bounds it. A tile of 128 x
// 128 brings 32 KB for 256 cycles of products, as many for an expert that has few of the 128 tokens.
#pragma once
#include <cuda.h>

#include "int8_tiles.cuh"

namespace i8 {

constexpr int kStageCols = 128;
constexpr int kMaxSplit = 8;
constexpr int kLinearThreads = 192;  // producer warp, tensor-core warp, four epilogue warps

struct LinearArgs {
  CUtensorMap w_map, x_map;
  const float* x_scale;
  const int32_t* x_sums;  // or NULL: no zero points
  RowsOf rows_of;
  fp4::Groups groups;     // row tiles: of 128 outputs
  void* y;
  int32_t rows, cols;     // of one expert's weight
  int32_t items;          // bound on the tiles
  int32_t split;          // blocks of a cluster that share a tile's K
  int32_t early;          // the codes are used where they are: loads of them need not wait for the launch before
  int32_t vec;            // rows of y start on 16-byte boundaries
};

template <int BN, int kCtas>
struct LinearShape {
  static constexpr int kW = kTileRows * kStageCols;
  static constexpr int kX = BN * kStageCols;
  static constexpr int kStage = kW + kX;
  static constexpr int kOut = 4 * 2048;  // 32 tokens x 32 outputs of each epilogue warp
  static constexpr int kTokens = BN * 8;  // the tile's token scales and sums
  static constexpr int kRoom = kSmemMax / kCtas - 2048 - kOut - kTokens;
  static constexpr int kStages = kRoom / kStage < 8 ? kRoom / kStage : 8;
  static constexpr int kSmem = kStages * kStage + kOut + kTokens + 1024 + 512;
  static constexpr int kAlloc = tmem_columns(2 * BN);  // two accumulators
  static_assert(2 * BN <= kAlloc && kAlloc * kCtas <= 512 && kStages >= 4, "the tile does not fit");
  static_assert(BN * kTileRows * 4 <= kStages * kStage, "a tile's sums have to fit in the stages");
};

// Persistent blocks. Roles run through the same tiles on their own: the producer and the tensor-core warp are up to two
// accumulators ahead of the epilogue.
template <int DT, int BN, int kCtas>
__global__ void __launch_bounds__(kLinearThreads, kCtas) linear_kernel(const __grid_constant__ LinearArgs p) {
  using S = LinearShape<BN, kCtas>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  uint8_t* out = smem + S::kStages * S::kStage;
  float* token_scale = reinterpret_cast<float*>(out + S::kOut);
  int32_t* token_sum = reinterpret_cast<int32_t*>(token_scale + BN);
  uint64_t* full = reinterpret_cast<uint64_t*>(token_sum + BN);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // this block's part of every tile's stages
  const int all = (p.cols + kStageCols - 1) / kStageCols;
  const int rank = p.split > 1 ? static_cast<int>(fp4::cluster_rank()) : 0;
  const int from = p.split > 1 ? all * rank / p.split : 0, to = p.split > 1 ? all * (rank + 1) / p.split : all, stages = to - from;
  const int first_item = p.split > 1 ? blockIdx.x / p.split : blockIdx.x, item_step = p.split > 1 ? gridDim.x / p.split : gridDim.x;
  TileAt t;
  bool have = first_item < p.items && fp4::find_tile(p.groups, first_item, BN, t);
  const auto next_tile = [&](int& id) {
    id += item_step;
    return id < p.items && fp4::find_tile(p.groups, id, BN, t);
  };
  if (warp == 0 && fp4::elect_one()) {
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
  }
  if (warp == 1) {
    pm::tmem_alloc(tmem_at, S::kAlloc);
    pm::tmem_relinquish();
  }
  pm::tc_fence_before();
  __syncthreads();
  fp4::grid_launch_dependents();  // after the allocation (launch.cuh)
  pm::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_at, 0);

  if (warp == 0) {
    fp4::Ring<S::kStages> ring;
    int it = 0;  // stages issued
    bool ok = true, waited = false;
    for (int id = first_item; ok && have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) continue;
      const int w_row = __shfl_sync(0xFFFFFFFFu, t.expert * p.rows + t.row_tile * kTileRows, 0);
      const int x_row = __shfl_sync(0xFFFFFFFFu, t.first, 0);
      const auto load_w = [&](int i, int s) {
        pm::mbar_arrive_expect_tx(&full[s], S::kStage);
        pm::tma_load_2d(smem + s * S::kStage, &p.w_map, i * kStageCols, w_row, &full[s]);
      };
      const auto load_x = [&](int i, int s) { pm::tma_load_2d(smem + s * S::kStage + S::kW, &p.x_map, i * kStageCols, x_row, &full[s]); };
      if (fp4::elect_one()) {
        int i = from;
        if (!waited) {
          // the first tile: the weight's part of every stage goes out before the tokens are quantised
          const int ahead = p.early ? min(stages, S::kStages) : 0;
          for (int j = 0; j < ahead; ++j) load_w(from + j, j);
          fp4::grid_wait();
          for (int j = 0; j < ahead; ++j, ++i, ++it, ring.next()) load_x(i, j);
        }
        for (; i < to; ++i, ++it, ring.next()) {
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
      ring.at(it);
    }
    if (!waited) fp4::grid_wait();  // no block ends before the launch it depends on
    // the last copies land before the block's shared memory goes, even if the tensor-core warp gave up
    for (int i = max(0, it - S::kStages); i < it; ++i)
      pm::mbar_wait(&full[i % S::kStages], (i / S::kStages) & 1, pm::kStatusTimeoutLoad);
    __syncwarp();
  } else if (warp == 1) {
    fp4::Ring<S::kStages> ring;
    int it = 0, n = 0;  // stages used, tiles begun
    bool ok = true;
    for (int id = first_item; ok && have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) continue;
      const int b = n & 1;
      const uint32_t d = tmem + b * BN;
      const uint32_t idesc = idesc_i8((static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, t.count, 0)) + 15u) & ~15u);
      if (fp4::elect_one()) {
        ok = n < 2 || pm::mbar_wait(&acc_empty[b], ((n >> 1) - 1) & 1, pm::kStatusTimeoutMma);
        pm::tc_fence_after();
        for (int i = from; ok && i < to; ++i, ++it, ring.next()) {
          ok = pm::mbar_wait(&full[ring.slot], ring.round, pm::kStatusTimeoutMma);
          if (!ok) break;
          pm::tc_fence_after();
          const uint32_t at = pm::smem_u32(smem) + ring.slot * S::kStage;
          const uint64_t a = pm::smem_desc_sw(at, 16, 1024, 2), x = pm::smem_desc_sw(at + S::kW, 16, 1024, 2);
          const int left = p.cols - i * kStageCols;  // columns behind the last are zeros
#pragma unroll
          for (int j = 0; j < kStageCols / 32; ++j)
            if (j * 32 < left) umma_i8(d, a + j * 2, x + j * 2, idesc, i != from || j != 0);
          pm::umma_commit(&empty[ring.slot]);
        }
        pm::umma_commit(&acc_full[b]);
      }
      __syncwarp();
      ++n;
      ok = __all_sync(0xFFFFFFFFu, ok);
      it = __reduce_max_sync(0xFFFFFFFFu, it);
      ring.at(it);
    }
    __syncwarp();
  } else {
    uint8_t* mine = out + (warp & 3) * 2048;
    const int thread = threadIdx.x - 64;
    int n = 0;
    fp4::grid_wait();  // the tokens' scales
    for (int id = first_item; have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) {
        if (rank == 0) zero_tile<DT>(p.y, t, p.rows, thread, 128);
        continue;
      }
      pm::named_bar_sync(1, 128);  // the last tile's are read
      for (int i = thread; i < BN; i += 128) {
        token_scale[i] = i < t.count ? p.x_scale[t.first + i] : 0.0f;
        token_sum[i] = i < t.count && p.x_sums != nullptr ? p.x_sums[t.first + i] : 0;
      }
      pm::named_bar_sync(1, 128);
      const int b = n & 1;
      const bool ok = pm::mbar_wait(&acc_full[b], (n >> 1) & 1, pm::kStatusTimeoutMma);
      if (!pm::named_bar_and(2, 128, ok)) break;
      pm::tc_fence_after();
      if (p.split > 1) {
        // one tile per cluster; its products are done, so the stages are free
        fp4::store_sums(tmem + b * BN, t, reinterpret_cast<float*>(smem));
        break;
      }
      store_tile<DT, true>(tmem + b * BN, p.y, t, p.rows, p.rows_of, static_cast<int64_t>(t.expert) * p.rows, token_scale, token_sum, 0, BN,
                           mine, p.vec != 0);
      pm::tc_fence_before();
      __syncwarp();
      if (lane == 0) pm::mbar_arrive(&acc_empty[b]);
      ++n;
    }
  }

  if (p.split > 1) {
    __syncwarp();
    fp4::cluster_sync();  // every block's sums are written
    if (fp4::find_tile(p.groups, first_item, BN, t) && t.expert != p.groups.experts)
      add_cluster_sums<DT, true>(reinterpret_cast<const float*>(smem), p.y, t, p.rows, p.rows_of, static_cast<int64_t>(t.expert) * p.rows,
                                 token_scale, token_sum, rank, p.split, kLinearThreads, p.vec != 0);
    __syncwarp();
    fp4::cluster_sync();  // nobody's shared memory goes while others read it
  }
  __syncthreads();
  if (warp == 1) {
    pm::tc_fence_after();
    pm::tmem_dealloc(tmem, S::kAlloc);
  }
}

}  // namespace i8
