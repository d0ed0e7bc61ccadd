// int8_few.cuh - the INT8 product of up to eight tokens and one weight, in one launch.
//
// The kernel is a stream of weight bytes: a tile of 128 outputs a block, or a share of its columns where a cluster of blocks
// splits them, by bulk tensor copies that wait for nothing but room. Meanwhile eight warps quantise the tokens, which every
// block needs, from L2: the maxima over whole rows, then the codes of the block's own columns into the tensor core's
// swizzled layout, eight rows of 128 columns a KB. The products take sixteen rows, the second eight of them the next KB:
// what they make of it goes into columns that nobody reads. Sums and their roundings are those of linear_kernel.
//
// 1 x 14336 x 4096 takes 13 us, 59 MB at 4.5 TB/s: the bytes are 9 us of it, the rest is the start and the last loads of 112
// blocks on 148 SMs.
#pragma once
#include "int8_linear.cuh"

namespace i8 {

constexpr int kFewTokens = 8;
constexpr int kFewWarps = 8;  // that quantise
constexpr int kFewThreads = 64 + 32 * kFewWarps;
constexpr int kFewRing = 12;  // most stages of the weight
constexpr int kFewHold = 2;   // units of its token that a lane keeps between the maximum and the codes
constexpr int kFewStage = kTileRows * kStageCols;
constexpr int kFewX = kFewTokens * kStageCols;  // the tokens' share of a stage
constexpr int kFewRest = kFewX + 4 * 2048 + 2 * 128 + 32 + 64 + 1024 + 512;  // KB after the last, epilogue, scales and sums, maxima, alignment, barriers

struct FewArgs {
  CUtensorMap w_map;
  const void* x;
  int64_t x_stride;
  RowsOf rows_of;
  void* y;
  int32_t tokens, rows, cols;
  int32_t split;  // blocks of a cluster that share a tile's columns
  int32_t x_stages;  // most stages of a block
  int32_t ring;   // stages of the weight under way
  int32_t vec;    // rows of y start on 16-byte boundaries
  int32_t x_vec;  // rows of x do, and have whole units
};

__host__ __device__ constexpr int few_smem(int x_stages, int ring) { return x_stages * kFewX + ring * kFewStage + kFewRest; }

template <int DT>
__global__ void __launch_bounds__(kFewThreads, 1) linear_few_kernel(const __grid_constant__ FewArgs p) {
  extern __shared__ uint8_t raw[];
  uint8_t* x = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  uint8_t* ring_at = x + (p.x_stages + 1) * kFewX;
  uint8_t* out = ring_at + p.ring * kFewStage;
  float* token_scale = reinterpret_cast<float*>(out + 4 * 2048);  // 32 of each, of which eight are used
  int32_t* token_sum = reinterpret_cast<int32_t*>(token_scale + 32);
  int32_t* token_total = token_sum + 32;  // over the cluster
  uint32_t* words = reinterpret_cast<uint32_t*>(token_total + kFewTokens);  // maxima, and sums of codes, of each warp
  uint64_t* full = reinterpret_cast<uint64_t*>(words + 2 * kFewWarps);
  uint64_t* empty = full + kFewRing;
  uint64_t* ready = empty + kFewRing;  // tokens are quantised
  uint64_t* done = ready + 1;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int all = (p.cols + kStageCols - 1) / kStageCols;
  const int rank = p.split > 1 ? static_cast<int>(fp4::cluster_rank()) : 0;
  const int from = all * rank / p.split, to = all * (rank + 1) / p.split;
  const TileAt t{0, static_cast<int32_t>(blockIdx.x) / p.split, 0, p.tokens, 0};
  // one, two, four or eight warps a token
  const int mine = warp - 2, each = p.tokens > 4 ? 1 : p.tokens > 2 ? 2 : p.tokens > 1 ? 4 : 8;
  const int token = max(mine, 0) / each, step = 32 * each, first = (max(mine, 0) % each) * 32 + lane;
  const bool has = mine >= 0 && token < p.tokens;
  const uint8_t* row = static_cast<const uint8_t*>(p.x) + (has ? token : 0) * p.x_stride * (DT == kF32 ? 4 : 2);
  const auto load = [&](int unit) {
    return p.x_vec != 0 ? load_unit<DT, true>(row, unit * kUnit, p.cols) : load_unit<DT, false>(row, unit * kUnit, p.cols);
  };
  const int units = (p.cols + kUnit - 1) / kUnit;
  fp4::grid_launch_dependents();
  if (warp == 0 && fp4::elect_one()) {
    pm::prefetch_tmap(&p.w_map);
    for (int s = 0; s < p.ring; ++s) {
      pm::mbar_init(&full[s], 1);
      pm::mbar_init(&empty[s], 1);
    }
    pm::mbar_init(ready, kFewWarps);
    pm::mbar_init(done, 1);
    pm::fence_mbar_init();
  }
  if (warp == 1) {
    pm::tmem_alloc(tmem_at, 32);
    pm::tmem_relinquish();
  }
  fp4::grid_wait();
  Unit<DT> held[kFewHold];
#pragma unroll
  for (int k = 0; k < kFewHold; ++k)
    if (has && first + k * step < units) held[k] = load(first + k * step);
  pm::tc_fence_before();
  __syncthreads();
  pm::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_at, 0);

  if (warp == 0) {
    int issued = 0;
    if (fp4::elect_one()) {
      int slot = 0;
      uint32_t parity = 0;
      for (int i = from; i < to; ++i) {
        if (issued >= p.ring && !pm::mbar_wait(&empty[slot], parity ^ 1u, pm::kStatusTimeoutLoad)) break;
        pm::mbar_arrive_expect_tx(&full[slot], kFewStage);
        pm::tma_load_2d(ring_at + slot * kFewStage, &p.w_map, i * kStageCols, t.row_tile * kTileRows, &full[slot]);
        ++issued;
        if (++slot == p.ring) {
          slot = 0;
          parity ^= 1u;
        }
      }
    }
    __syncwarp();
    issued = __reduce_max_sync(0xFFFFFFFFu, issued);
    // the last copies land before the block's shared memory goes, even if the tensor-core warp gave up
    for (int i = max(0, issued - p.ring); i < issued; ++i) pm::mbar_wait(&full[i % p.ring], (i / p.ring) & 1, pm::kStatusTimeoutLoad);
    __syncwarp();
  } else if (warp == 1) {
    if (fp4::elect_one()) {
      constexpr uint32_t kIdesc = idesc_i8(16);
      bool ok = pm::mbar_wait(ready, 0, pm::kStatusTimeoutMma);
      int slot = 0;
      uint32_t parity = 0;
      for (int i = from; ok && i < to; ++i) {
        ok = pm::mbar_wait(&full[slot], parity, pm::kStatusTimeoutMma);
        if (!ok) break;
        pm::tc_fence_after();
        const uint64_t a = pm::smem_desc_sw(pm::smem_u32(ring_at) + slot * kFewStage, 16, 1024, 2);
        const uint64_t b = pm::smem_desc_sw(pm::smem_u32(x) + (i - from) * kFewX, 16, 1024, 2);
        const int left = p.cols - i * kStageCols;  // the weight's columns behind the last are zeros
#pragma unroll
        for (int j = 0; j < kStageCols / 32; ++j)
          if (j * 32 < left) umma_i8(tmem, a + j * 2, b + j * 2, kIdesc, i != from || j != 0);
        pm::umma_commit(&empty[slot]);
        if (++slot == p.ring) {
          slot = 0;
          parity ^= 1u;
        }
      }
      pm::umma_commit(done);
    }
    __syncwarp();
  } else {
    uint32_t top = 0u;
    if (has) {
#pragma unroll
      for (int k = 0; k < kFewHold; ++k)
        if (first + k * step < units) top = max(top, unit_top<DT>(held[k]));
      for (int u = first + kFewHold * step; u < units; u += step) top = max(top, unit_top<DT>(load(u)));
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (lane == 0) words[mine] = top;
    pm::named_bar_sync(1, 32 * kFewWarps);
    for (int k = 0; k < each; ++k) top = max(top, words[token * each + k]);
    const Quotient q = quotient_of(top);
    int sum = 0;
    const int begin = from * (kStageCols / kUnit), end = min(units, to * (kStageCols / kUnit));
    const auto write = [&](int u, const Unit<DT>& unit) {
      const int in = u - begin;
      uint8_t* at = x + (in >> 3) * kFewX + token * kStageCols + (((in & 7) ^ token) << 4);
      sum += store_codes<DT>(unit, q, reinterpret_cast<int8_t*>(at));
    };
    if (has) {
#pragma unroll
      for (int k = 0; k < kFewHold; ++k) {
        const int u = first + k * step;
        if (u >= begin && u < end) write(u, held[k]);
      }
      for (int u = first + kFewHold * step; u < end; u += step)
        if (u >= begin) write(u, load(u));
    }
    pm::fence_proxy_async_smem();
    sum = __reduce_add_sync(0xFFFFFFFFu, sum);
    if (lane == 0) {
      pm::mbar_arrive(ready);
      words[kFewWarps + mine] = static_cast<uint32_t>(sum);
      if (has && mine % each == 0) token_scale[token] = q.scale;
    }
    pm::named_bar_sync(1, 32 * kFewWarps);
    if (const int i = threadIdx.x - 64; i < 32) {
      int total = 0;
      if (i < p.tokens)
        for (int k = 0; k < each; ++k) total += static_cast<int>(words[kFewWarps + i * each + k]);
      token_sum[i] = total;  // of this block's columns
      if (i >= p.tokens) token_scale[i] = 0.0f;
    }
    pm::named_bar_sync(1, 32 * kFewWarps);
    if (warp < 6 && __all_sync(0xFFFFFFFFu, pm::mbar_wait(done, 0, pm::kStatusTimeoutMma))) {
      pm::tc_fence_after();
      if (p.split > 1) fp4::store_sums(tmem, t, reinterpret_cast<float*>(ring_at));  // the products are done, so the ring is free
      else store_tile<DT, true>(tmem, p.y, t, p.rows, p.rows_of, 0, token_scale, token_sum, 0, kFewTokens, out + (warp & 3) * 2048, p.vec != 0);
      pm::tc_fence_before();
    }
  }

  if (p.split > 1) {
    __syncwarp();
    fp4::cluster_sync();  // every block's sums are written
    if (threadIdx.x < kFewTokens / 4) {
      // the tokens' sums of codes over all columns
      int4 total = make_int4(0, 0, 0, 0);
      for (int r = 0; r < p.split; ++r) {
        const float4 v = fp4::load_cluster(pm::smem_u32(token_sum) + threadIdx.x * 16, static_cast<uint32_t>(r));
        total.x += __float_as_int(v.x);
        total.y += __float_as_int(v.y);
        total.z += __float_as_int(v.z);
        total.w += __float_as_int(v.w);
      }
      reinterpret_cast<int4*>(token_total)[threadIdx.x] = total;
    }
    __syncthreads();
    add_cluster_sums<DT, true>(reinterpret_cast<const float*>(ring_at), p.y, t, p.rows, p.rows_of, 0, token_scale, token_total, rank, p.split,
                               kFewThreads, p.vec != 0);
    __syncwarp();
    fp4::cluster_sync();  // nobody's shared memory goes while others read it
  }
  __syncthreads();
  if (warp == 1) {
    pm::tc_fence_after();
    pm::tmem_dealloc(tmem, 32);
  }
}

}  // namespace i8
