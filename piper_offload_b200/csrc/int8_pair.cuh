// int8_pair.cuh - the INT8 product on pairs of SMs (cta_group::2): tiles of 256 outputs x up to 256 tokens.
//
// On one SM a step of 32 columns brings 4 KB of the weight and 8 KB of tokens into shared memory and reads them again for
// 128 cycles of products: 24 KB at 128 bytes a cycle, 192 cycles, and that is what a step takes (4096 x 14336 x 4096: 164 us
// in tiles of 128 x 256). In a pair each SM holds 128 rows of the weight and half of the tokens, which the tensor cores of
// both read: 16 KB for the same 128 cycles. 4096 x 14336 x 4096 then takes 154 us with the launch before (10), the tensor
// pipe active for 92 % of the product while the power limit holds the clock at 1.6 GHz (3.3 POP/s); 184 to 189 us in a program.
//
// The even block of a pair issues the products for both; each block loads its own halves, counted on the even block's
// barrier, and has its own 128 outputs in its tensor memory. Finished products are announced to both blocks.
#pragma once
#include "int8_linear.cuh"

namespace i8 {

template <int BN>
struct PairShape {
  static constexpr int kW = kTileRows * kStageCols;
  static constexpr int kX = BN / 2 * kStageCols;
  static constexpr int kStage = kW + kX;
  static constexpr int kOut = 4 * 2048;
  static constexpr int kTokens = BN * 8;
  static constexpr int kRoom = kSmemMax - 2048 - kOut - kTokens;
  static constexpr int kStages = kRoom / kStage < 8 ? kRoom / kStage : 8;
  static constexpr int kSmem = kStages * kStage + kOut + kTokens + 1024 + 512;
  static constexpr int kAlloc = tmem_columns(2 * BN);  // two accumulators
  static_assert(2 * BN <= kAlloc && kStages >= 4, "the tile does not fit");
};

// signed 8-bit operands, both K-major, 32-bit sums, M = 256.
__host__ __device__ constexpr uint32_t idesc_i8_pair(uint32_t n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((256u >> 4) << 24); }

__device__ __forceinline__ void umma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Persistent pairs of blocks (a cluster of two). Row tiles: of 256 outputs.
template <int DT, int BN>
__global__ void __launch_bounds__(kLinearThreads, 1) linear_pair_kernel(const __grid_constant__ LinearArgs p) {
  using S = PairShape<BN>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  uint8_t* out = smem + S::kStages * S::kStage;
  float* token_scale = reinterpret_cast<float*>(out + S::kOut);
  int32_t* token_sum = reinterpret_cast<int32_t*>(token_scale + BN);
  uint64_t* full = reinterpret_cast<uint64_t*>(token_sum + BN);  // both blocks' halves landed (the even block's counts)
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + 2;  // both blocks' epilogues have read it (the even block's counts)
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = fp4::cluster_rank();
  const int stages = (p.cols + kStageCols - 1) / kStageCols;
  const int first_item = blockIdx.x / 2, item_step = gridDim.x / 2;
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
      pm::mbar_init(&acc_empty[b], 8);
    }
    pm::fence_mbar_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_at, S::kAlloc);
  pm::tc_fence_before();
  __syncthreads();
  fp4::grid_launch_dependents();  // after the allocation (launch.cuh)
  fp4::cluster_sync();  // both blocks' barriers are there
  pm::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_at, 0);
  // the tokens that a tile's products take: in thirty-twos, half of them this block's
  const auto computed = [](int count) { return (static_cast<uint32_t>(count) + 31u) & ~31u; };

  if (warp == 0) {
    fp4::Ring<S::kStages> ring;
    int it = 0;  // stages issued
    bool ok = true, waited = false;
    for (int id = first_item; ok && have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) continue;
      const int w_row = __shfl_sync(0xFFFFFFFFu, t.expert * p.rows + t.row_tile * 2 * kTileRows + static_cast<int>(rank) * kTileRows, 0);
      const int x_row = __shfl_sync(0xFFFFFFFFu, t.first + static_cast<int>(rank * computed(t.count) / 2), 0);
      const auto load_w = [&](int i, int s) {
        if (rank == 0) pm::mbar_arrive_expect_tx(&full[s], 2 * S::kStage);
        tma_load_2d_pair(smem + s * S::kStage, &p.w_map, i * kStageCols, w_row, in_block(pm::smem_u32(&full[s]), 0));
      };
      const auto load_x = [&](int i, int s) {
        tma_load_2d_pair(smem + s * S::kStage + S::kW, &p.x_map, i * kStageCols, x_row, in_block(pm::smem_u32(&full[s]), 0));
      };
      if (fp4::elect_one()) {
        int i = 0;
        if (!waited) {
          // the first tile: the weight's part of every stage goes out before the tokens are quantised
          const int ahead = p.early ? min(stages, S::kStages) : 0;
          for (int j = 0; j < ahead; ++j) load_w(j, j);
          fp4::grid_wait();
          for (int j = 0; j < ahead; ++j, ++i, ++it, ring.next()) load_x(i, j);
        }
        for (; i < stages; ++i, ++it, ring.next()) {
          ok = it < S::kStages || mbar_wait_pair(&empty[ring.slot], ring.round ^ 1u, pm::kStatusTimeoutLoad);
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
    // the last copies of both blocks land before either's shared memory goes, even if the tensor-core warp gave up
    if (rank == 0)
      for (int i = max(0, it - S::kStages); i < it; ++i)
        mbar_wait_pair(&full[i % S::kStages], (i / S::kStages) & 1, pm::kStatusTimeoutLoad);
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    fp4::Ring<S::kStages> ring;
    int it = 0, n = 0;  // stages used, tiles begun
    bool ok = true;
    for (int id = first_item; ok && have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) continue;
      const int b = n & 1;
      const uint32_t d = tmem + b * BN;
      const uint32_t idesc = idesc_i8_pair(computed(__shfl_sync(0xFFFFFFFFu, t.count, 0)));
      if (fp4::elect_one()) {
        ok = n < 2 || mbar_wait_pair(&acc_empty[b], ((n >> 1) - 1) & 1, pm::kStatusTimeoutMma);
        pm::tc_fence_after();
        for (int i = 0; ok && i < stages; ++i, ++it, ring.next()) {
          ok = mbar_wait_pair(&full[ring.slot], ring.round, pm::kStatusTimeoutMma);
          if (!ok) break;
          pm::tc_fence_after();
          const uint32_t at = pm::smem_u32(smem) + ring.slot * S::kStage;
          const uint64_t a = pm::smem_desc_sw(at, 16, 1024, 2), x = pm::smem_desc_sw(at + S::kW, 16, 1024, 2);
          const int left = p.cols - i * kStageCols;  // columns behind the last are zeros
#pragma unroll
          for (int j = 0; j < kStageCols / 32; ++j)
            if (j * 32 < left) umma_i8_pair(d, a + j * 2, x + j * 2, idesc, i != 0 || j != 0);
          umma_commit_pair(&empty[ring.slot]);
        }
        umma_commit_pair(&acc_full[b]);
      }
      __syncwarp();
      ++n;
      ok = __all_sync(0xFFFFFFFFu, ok);
      it = __reduce_max_sync(0xFFFFFFFFu, it);
      ring.at(it);
    }
    __syncwarp();
  } else if (warp >= 2) {
    uint8_t* mine = out + (warp & 3) * 2048;
    const int thread = threadIdx.x - 64;
    int n = 0;
    fp4::grid_wait();  // the tokens' scales
    for (int id = first_item; have; have = next_tile(id)) {
      TileAt half = t;  // this block's outputs
      half.row_tile = t.row_tile * 2 + static_cast<int>(rank);
      if (t.expert == p.groups.experts) {
        zero_tile<DT>(p.y, half, p.rows, thread, 128);
        continue;
      }
      pm::named_bar_sync(1, 128);  // the last tile's are read
      for (int i = thread; i < BN; i += 128) {
        token_scale[i] = i < t.count ? p.x_scale[t.first + i] : 0.0f;
        token_sum[i] = i < t.count && p.x_sums != nullptr ? p.x_sums[t.first + i] : 0;
      }
      pm::named_bar_sync(1, 128);
      const int b = n & 1;
      const bool ok = mbar_wait_pair(&acc_full[b], (n >> 1) & 1, pm::kStatusTimeoutMma);
      if (!pm::named_bar_and(2, 128, ok)) break;
      pm::tc_fence_after();
      store_tile<DT, true>(tmem + b * BN, p.y, half, p.rows, p.rows_of, static_cast<int64_t>(t.expert) * p.rows, token_scale, token_sum, 0, BN,
                           mine, p.vec != 0);
      pm::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_pair(in_block(pm::smem_u32(&acc_empty[b]), 0));
      ++n;
    }
  }

  __syncwarp();
  fp4::cluster_sync();  // nobody's shared or tensor memory goes while the other block uses it
  if (warp == 1) {
    pm::tc_fence_after();
    tmem_dealloc_pair(tmem, S::kAlloc);
  }
}

}  // namespace i8
