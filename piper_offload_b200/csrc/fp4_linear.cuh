// fp4_linear.cuh - y[t, n] = alpha * sum_k x[t, k] * w[n, k] with both operands in packed FP4.
//
// The weight's rows are the tensor core's 128-row operand and the tokens its
// N side, so a tile is 128 outputs x up to BN tokens and the instruction's N
// follows the tokens that are there: experts with few rows waste little.
// A K step is 64 values (32 bytes a row). Codes come by bulk tensor copies in
// the 128-byte swizzle (256 values a row and stage); block scales reach shared
// memory as 512-byte tiles of the swizzled layout and go on to tensor memory
// by tcgen05.cp ahead of the products that use them. The scales are applied
// inside the tensor core; sums are fp32 in tensor memory, and the one rounding
// is that of the output.
//
// Many tokens: their codes and scales are made by a launch before (prepare_kernel),
// tiles are 32, 128 or 192 tokens wide. A handful (kFused): the kernel is a
// stream of weight bytes, so four warps quantize the tokens on the way, each
// every fourth stage, there is no launch before, and two blocks share an SM, one
// starting or ending while the other streams. Where there are too few tiles for
// the SMs, a cluster of blocks splits K; each leaves its sums in its own shared
// memory and every block adds up its share of the tokens over the cluster, in
// rank order, so that results do not depend on timing.
//
// Times on a B200, whole calls back to back at 1965 MHz, and what bounds them.
// Few tokens: HBM, after about 5 us of launch and first loads; 1 x 14336 x 4096
// NVFP4 9.6 us (3.5 TB/s; called from a program 10.3), x 28672 14.5 (4.6), 16 tokens
// over 8 experts of 14336 x 4096 two-level 38.0 us (5.2 TB/s). Many: not known.
// 4096 x 14336 x 4096, the tokens' quantisation included, takes 135 us in NVFP4
// (3.6 PFLOP/s, the pipe 43 % active; 164 us in a running program, under the power
// cap) and 117 in MXFP4 (4.1), which has half the scales and a buffer of them in
// tensor memory for each stage, where NVFP4 has two for four stages. What a step of
// 64 values brings into shared memory and out again, 11.5 KB each at 128 bytes a
// cycle, would take more than the 170 to 176 cycles measured, so that account does
// not hold. 2048 x 4096 x 4096 MXFP4 26 us (2.6 PFLOP/s). Wider tiles do not fit
// beside two accumulators; 256 x 192 over a pair of SMs took 226 us.
//
// Weight scales in rows are read by one warp, in pieces as wide as their count a
// row allows. In single bytes or pairs that warp sets the pace: 1 x 4096 x 2880
// MXFP4 (90 scales a row) 23.5 us, 6.1 from swizzled tiles; 333 tokens 25.4 and
// 9.6; x 2896 NVFP4 (181) 55 and 20. With 128 scales a row 8.5 and 7.
#pragma once
#include <cuda.h>

#include "fp4_ptx.cuh"
#include "fp4_quant.cuh"
#include "fp4_tiles.cuh"

namespace fp4 {

constexpr int kStageCols = 256;      // K values per stage
constexpr int kStageBytes = kStageCols / 2;
constexpr int kQuantWarps = 4;       // kFused
constexpr int kFusedCtas = 2;        // kFused: blocks per SM
constexpr int kMaxSplit = 8;

// Where the weight's scales come from: whole swizzled tiles by bulk copies, or
// by a warp that reads them (swizzled tiles with columns that do not exist, or
// rows) in pieces of 16 / 8 / 4 / 1 bytes.
enum : int { kScalesBulk = 0, kScalesTiles = 1, kScalesRows = 2 };

struct LinearArgs {
  CUtensorMap w_map, x_map;
  const uint8_t* w_scale;
  const uint8_t* x_scale;  // swizzled tiles, rows as first_scale_row places them (not kFused)
  const float* w_second;   // (experts) or NULL
  const float* x_second;   // one or NULL
  const void* x;           // the tokens themselves (kFused)
  int64_t x_stride;
  Groups groups;           // row tiles: of 128 outputs
  void* y;
  int32_t rows, cols;      // of one expert's weight
  int32_t k_steps;         // of 64 values
  int32_t scale_tiles;     // tiles of 4 scales per row (weight and tokens alike)
  int32_t items;           // bound on the tiles
  int32_t split;           // blocks of a cluster that share a tile's K
  int32_t early;           // the codes are used where they are: loads of them need not wait for the launch before
  int32_t vec;             // rows of y start on 16-byte boundaries
  int32_t x_vec;           // rows of x start on 32-byte boundaries
  int32_t scale_mode;      // of the tokens
  int32_t scale_source;    // kScales...
  int32_t scale_cols;      // scales per row (kScalesRows)
  int32_t scale_piece;     // bytes of an aligned load of the weight's scales
};

template <int FMT, int BN, bool kFused>
struct LinearShape {
  static constexpr int kTiles = FMT == kNV ? 4 : 2;                 // scale tiles per stage and 128 rows
  static constexpr int kCtas = kFused ? kFusedCtas : 1;             // per SM
  static constexpr int kXBlocks = (BN + 127) / 128;                 // 128-token scale blocks per tile
  static constexpr int kW = kTileRows * kStageBytes;
  static constexpr int kX = BN * kStageBytes;
  static constexpr int kSW = kTiles * 512;
  static constexpr int kSX = kXBlocks * kTiles * 512;
  static constexpr int kStage = kW + kX + kSW + kSX;
  static constexpr int kOut = 4 * 2048;                             // 32 tokens x 32 outputs of each epilogue warp
  static constexpr int kRoom = kSmemMax / kCtas - 2048 - kOut;
  static constexpr int kStages = kRoom / kStage < 8 ? kRoom / kStage : 8;
  static constexpr int kSmem = kStages * kStage + kOut + 1024 + 512;
  static constexpr bool kCanSplit = BN * kTileRows * 4 <= kStages * kStage;
  // tensor memory: two accumulators, then buffers of scales, one per stage if they fit
  static constexpr int kScaleCols = kTiles * 4 * (1 + kXBlocks);
  static constexpr int kBufs = (512 / kCtas - 2 * BN) / kScaleCols < kStages ? (512 / kCtas - 2 * BN) / kScaleCols : kStages;
  static constexpr int kCols = 2 * BN + kBufs * kScaleCols;
  // with fewer buffers than stages the copies of scales wait for products, and get a warp of their own: 4096 tokens x
  // 14336 x 4096 NVFP4 136 us against 145; with a buffer per stage one warp does both, 6 to 10 % faster on small calls
  static constexpr bool kCopyWarp = kBufs < kStages;
  static constexpr int kFirstQuantWarp = kCopyWarp ? 8 : 7;
  static constexpr int kThreads = 32 * kFirstQuantWarp + (kFused ? 32 * kQuantWarps : 0);
  static constexpr int kAlloc = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kAlloc * kCtas <= 512 && kStages >= 4 && kBufs >= 2, "the tile does not fit");
  // a warp's next stage is at most one round of the ring away: further, a wait on a slot's parity could pass a round early
  static_assert(!kFused || kQuantWarps <= kStages, "more quantising warps than stages");
};

// The scales that one stage needs of the weight: 128 rows x kTiles words, four rows a lane.
template <int FMT>
struct ScaleWords {
  static constexpr int kTiles = FMT == kNV ? 4 : 2;
  uint32_t w[4][kTiles];
};

template <int FMT>
__device__ __forceinline__ ScaleWords<FMT> load_scale_words(const LinearArgs& p, const TileAt& t, int stage, int lane) {
  constexpr int kTiles = ScaleWords<FMT>::kTiles;
  constexpr int kBytes = 4 * kTiles;
  ScaleWords<FMT> s;
  const int tile0 = stage * kTiles;
  if (p.scale_source == kScalesTiles) {
    // a lane's 16 bytes of a tile are its four rows' words
    const uint8_t* from = p.w_scale + ((static_cast<int64_t>(t.expert) * p.groups.row_tiles + t.row_tile) * p.scale_tiles + tile0) * 512 + lane * 16;
#pragma unroll
    for (int k = 0; k < kTiles; ++k) {
      uint32_t v[4] = {0u, 0u, 0u, 0u};
      const int left = p.scale_cols - (tile0 + k) * 4;  // scales of this tile that exist
      if (left > 0) {
        if (p.scale_piece >= 16) {
          const uint4 q = *reinterpret_cast<const uint4*>(from + k * 512);
          v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        } else {
#pragma unroll
          for (int b = 0; b < 16; ++b) v[b >> 2] |= static_cast<uint32_t>(from[k * 512 + b]) << (8 * (b & 3));
        }
      }
      const uint32_t mask = left >= 4 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
#pragma unroll
      for (int j = 0; j < 4; ++j) s.w[j][k] = v[j] & mask;
    }
    return s;
  }
  const int c0 = tile0 * 4, bytes = min(kBytes, p.scale_cols - c0);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int k = 0; k < kTiles; ++k) s.w[j][k] = 0u;
    const int row = t.row_tile * kTileRows + j * 32 + lane;
    if (row >= p.rows) continue;
    const uint8_t* from = p.w_scale + (static_cast<int64_t>(t.expert) * p.rows + row) * p.scale_cols + c0;
    if (bytes == kBytes && p.scale_piece >= kBytes) {
      if constexpr (kBytes == 16) {
        const uint4 q = *reinterpret_cast<const uint4*>(from);
        s.w[j][0] = q.x; s.w[j][1] = q.y; s.w[j][2] = q.z; s.w[j][3] = q.w;
      } else {
        const uint2 q = *reinterpret_cast<const uint2*>(from);
        s.w[j][0] = q.x; s.w[j][1] = q.y;
      }
    } else if (p.scale_piece >= 4 && bytes % 4 == 0) {
#pragma unroll
      for (int k = 0; k < kTiles; ++k)
        if (k * 4 < bytes) s.w[j][k] = *reinterpret_cast<const uint32_t*>(from + k * 4);
    } else {
#pragma unroll
      for (int b = 0; b < kBytes; ++b)
        if (b < bytes) s.w[j][b >> 2] |= static_cast<uint32_t>(from[b]) << (8 * (b & 3));
    }
  }
  return s;
}

// Two tokens of a stage, as a warp holds them: half a warp a row.
template <int DT>
using TokenBlock = Raw<DT>;

template <int DT>
__device__ __forceinline__ TokenBlock<DT> load_tokens(const LinearArgs& p, const TileAt& t, int stage, int row0) {
  const int lane = threadIdx.x & 31;
  const int col = stage * kStageCols + (lane & 15) * kUnit;
  const int r = row0 + (lane >> 4);
  if (r < t.count && col < p.cols) return load_unit<DT>(p.x, (t.first + r) * p.x_stride + col, p.x_vec != 0);
  return TokenBlock<DT>{};
}

// A warp quantizes them into the operand's swizzled rows and its scale tiles.
template <int DT, int FMT>
__device__ __forceinline__ void quantize_tokens(const LinearArgs& p, const TileAt& t, const TokenBlock<DT>& b, int stage, int row0,
                                                uint8_t* codes, uint8_t* scales, const Second& second) {
  const int lane = threadIdx.x & 31, unit = lane & 15;
  const bool in_cols = stage * kStageCols + unit * kUnit < p.cols;
  const int r = row0 + (lane >> 4);
  float v[16];
  to_floats(b, v);
  const Coded c = quantize16<FMT>(v, p.scale_mode, second);
  const uint32_t word = gather_scales<FMT>(in_cols ? c.byte : 0u);
  if (r < t.count) {
    *reinterpret_cast<uint2*>(codes + r * kStageBytes + (((unit >> 1) ^ (r & 7)) << 4) + (unit & 1) * 8) = c.codes;
    constexpr int kLanes = FMT == kNV ? 4 : 8;  // units per scale tile
    if (unit % kLanes == 0) *reinterpret_cast<uint32_t*>(scales + (unit / kLanes) * 512 + (r & 31) * 16 + (r >> 5) * 4) = word;
  }
}

// Persistent blocks. Roles run through the same tiles on their own: the
// producers and the tensor-core warp are up to two accumulators ahead of the
// epilogue.
template <int DT, int FMT, int BN, bool kFused>
__global__ void __launch_bounds__(LinearShape<FMT, BN, kFused>::kThreads, LinearShape<FMT, BN, kFused>::kCtas)
    linear_kernel(const __grid_constant__ LinearArgs p) {
  using S = LinearShape<FMT, BN, kFused>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  uint8_t* out = smem + S::kStages * S::kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(out + S::kOut);
  uint64_t* empty = full + S::kStages;
  uint64_t* scales_in = empty + S::kStages;  // a buffer of scales is in tensor memory
  uint64_t* acc_full = scales_in + S::kBufs;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // this block's part of every tile's stages
  const int all = (p.k_steps + 3) / 4;
  const int rank = p.split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int from = p.split > 1 ? all * rank / p.split : 0, to = p.split > 1 ? all * (rank + 1) / p.split : all, stages = to - from;
  const int first_item = p.split > 1 ? blockIdx.x / p.split : blockIdx.x, item_step = p.split > 1 ? gridDim.x / p.split : gridDim.x;
  const bool bulk = p.scale_source == kScalesBulk;
  // every warp finds the first tile, and has its first loads under way, while the barriers and tensor memory are set up
  TileAt t;
  bool have = first_item < p.items && find_tile(p.groups, first_item, BN, t);
  const auto next_tile = [&](int& id) {
    id += item_step;
    return id < p.items && find_tile(p.groups, id, BN, t);
  };
  TokenBlock<DT> first_tokens;  // kFused: of this quantising warp's first stage
  if constexpr (kFused)
    if (warp >= S::kFirstQuantWarp && have && t.expert != p.groups.experts && from + warp - S::kFirstQuantWarp < to)
      first_tokens = load_tokens<DT>(p, t, from + warp - S::kFirstQuantWarp, 0);
  if (warp == 0 && elect_one()) {
    for (int s = 0; s < S::kStages; ++s) {
      pm::mbar_init(&full[s], 1 + (p.scale_source != kScalesBulk) + kFused);
      pm::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < S::kBufs; ++b) pm::mbar_init(&scales_in[b], 1);
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
  pm::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_at, 0);
  // the scales of stage i from shared to tensor memory
  const auto copy_scales = [&](int i, int slot, int buf) {
    const uint32_t at = pm::smem_u32(smem) + slot * S::kStage;
    const uint32_t sw = tmem + 2 * BN + buf * S::kScaleCols, sx = sw + S::kTiles * 4;
    const int tiles = p.scale_tiles - i * S::kTiles;
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
  };

  if (warp == 0) {
    Ring<S::kStages> ring;
    int it = 0;  // stages issued
    bool ok = true, waited = false;
    for (int id = first_item; ok && have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) continue;
      const int w_row = __shfl_sync(0xFFFFFFFFu, t.expert * p.rows + t.row_tile * kTileRows, 0);
      const int x_row = __shfl_sync(0xFFFFFFFFu, t.first, 0);
      const uint8_t* w_scale =
          p.w_scale + static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, t.expert * p.groups.row_tiles + t.row_tile, 0)) * p.scale_tiles * 512;
      const uint8_t* x_scale = p.x_scale + static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, t.scale_row >> 7, 0)) * p.scale_tiles * 512;
      const auto load_w = [&](int i, int s) {
        uint8_t* at = smem + s * S::kStage;
        const int tiles = min(S::kTiles, p.scale_tiles - i * S::kTiles);
        pm::mbar_arrive_expect_tx(&full[s], S::kW + (kFused ? 0 : S::kX) + tiles * 512 * ((bulk ? 1 : 0) + (kFused ? 0 : S::kXBlocks)));
        pm::tma_load_2d(at, &p.w_map, i * kStageBytes, w_row, &full[s]);
        if (bulk) pm::bulk_g2s(at + S::kW + S::kX, w_scale + static_cast<int64_t>(i) * S::kTiles * 512, tiles * 512, &full[s]);
      };
      const auto load_x = [&](int i, int s) {
        if constexpr (!kFused) {
          uint8_t* at = smem + s * S::kStage;
          const int tiles = min(S::kTiles, p.scale_tiles - i * S::kTiles);
          pm::tma_load_2d(at + S::kW, &p.x_map, i * kStageBytes, x_row, &full[s]);
#pragma unroll
          for (int b = 0; b < S::kXBlocks; ++b)
            pm::bulk_g2s(at + S::kW + S::kX + S::kSW + b * S::kTiles * 512,
                         x_scale + (static_cast<int64_t>(b) * p.scale_tiles + i * S::kTiles) * 512, tiles * 512, &full[s]);
        }
      };
      if (elect_one()) {
        int i = from;
        if (!waited) {
          // the first tile: the weight's part of every stage goes out before the tokens are quantized
          const int ahead = p.early ? min(stages, S::kStages) : 0;
          for (int j = 0; j < ahead; ++j) load_w(from + j, j);
          grid_wait();
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
    if (!waited) grid_wait();  // no block ends before the launch it depends on
    // the last copies land before the block's shared memory goes, even if the tensor-core warp gave up
    for (int i = max(0, it - S::kStages); i < it; ++i)
      pm::mbar_wait(&full[i % S::kStages], (i / S::kStages) & 1, pm::kStatusTimeoutLoad);
    __syncwarp();
  } else if (warp == 1) {
    Ring<S::kStages> ring;
    Ring<S::kBufs> buf;
    int it = 0, n = 0;  // stages used, tiles begun
    bool ok = true;
    for (int id = first_item; ok && have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) continue;
      const int b = n & 1;
      const uint32_t d = tmem + b * BN;
      const uint32_t n_mma = (static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, t.count, 0)) + 15u) & ~15u;  // computed token columns
      const uint32_t idesc = idesc_fp4(kTileRows, n_mma, FMT == kMX, 0);
      if (elect_one()) {
        ok = n < 2 || pm::mbar_wait(&acc_empty[b], ((n >> 1) - 1) & 1, pm::kStatusTimeoutMma);
        pm::tc_fence_after();
        for (int i = from; ok && i < to; ++i, ++it, ring.next(), buf.next()) {
          ok = pm::mbar_wait(&full[ring.slot], ring.round, pm::kStatusTimeoutMma);
          if (S::kCopyWarp) ok = ok && pm::mbar_wait(&scales_in[buf.slot], buf.round, pm::kStatusTimeoutMma);
          if (!ok) break;
          pm::tc_fence_after();
          if (!S::kCopyWarp) copy_scales(i, ring.slot, buf.slot);
          const uint32_t at = pm::smem_u32(smem) + ring.slot * S::kStage;
          const uint32_t sw = tmem + 2 * BN + buf.slot * S::kScaleCols, sx = sw + S::kTiles * 4;
          const int steps = p.k_steps - i * 4;
          const uint64_t a = pm::smem_desc_sw(at, 16, 1024, 2), x = pm::smem_desc_sw(at + S::kW, 16, 1024, 2);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            constexpr uint32_t kSecondHalf = (2u << 4) | (2u << 29);  // scale bytes 2 and 3 of a column
            const uint32_t tile = FMT == kNV ? j : j >> 1;
            if (j < steps)
              umma_fp4<FMT>(d, a + j * 2, x + j * 2, FMT == kMX && (j & 1) ? idesc | kSecondHalf : idesc, sw + tile * 4,
                            sx + tile * 4 * S::kXBlocks, i != from || j != 0);
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
      ring.at(it);
      buf.at(it);
    }
    __syncwarp();
  } else if (S::kCopyWarp && warp == 7) {
    // scales from shared to tensor memory: up to twelve copies a stage, which take their issuer as long as the products
    Ring<S::kStages> ring, old;  // this stage; the one kBufs stages ago
    Ring<S::kBufs> buf;
    int it = 0;
    bool ok = true;
    for (int id = first_item; ok && have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) continue;
      if (elect_one()) {
        for (int i = from; i < to; ++i, ++it, ring.next(), buf.next()) {
          if (S::kBufs < S::kStages && it >= S::kBufs) {
            // the buffer's last readers have finished
            ok = pm::mbar_wait(&empty[old.slot], old.round, pm::kStatusTimeoutMma);
            old.next();
          }
          ok = ok && pm::mbar_wait(&full[ring.slot], ring.round, pm::kStatusTimeoutMma);
          if (!ok) break;
          pm::tc_fence_after();
          copy_scales(i, ring.slot, buf.slot);
          pm::umma_commit(&scales_in[buf.slot]);
        }
      }
      __syncwarp();
      ok = __all_sync(0xFFFFFFFFu, ok);
      it = __reduce_max_sync(0xFFFFFFFFu, it);
      ring.at(it);
      buf.at(it);
      old.at(max(it - S::kBufs, 0));
    }
    __syncwarp();
  } else if (warp < 6) {
    const float x_second = p.x_second != nullptr ? *p.x_second : 1.0f;
    uint8_t* mine = out + (warp & 3) * 2048;
    int n = 0;
    for (int id = first_item; have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) {
        if (rank == 0) store_zeros<DT>(p.y, t, p.rows, threadIdx.x - 64, 128);
        continue;
      }
      const int b = n & 1;
      const bool ok = pm::mbar_wait(&acc_full[b], (n >> 1) & 1, pm::kStatusTimeoutMma);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      pm::tc_fence_after();
      if (S::kCanSplit && p.split > 1) {
        // one tile per cluster; its products are done, so the stages are free
        store_sums(tmem + b * BN, t, reinterpret_cast<float*>(smem));
        break;
      }
      const float alpha = (p.w_second != nullptr ? p.w_second[t.expert] : 1.0f) * x_second;
      store_tile<DT>(tmem + b * BN, p.y, t, p.rows, alpha, 0, BN, mine, p.vec != 0);
      pm::tc_fence_before();
      __syncwarp();
      if (lane == 0) pm::mbar_arrive(&acc_empty[b]);
      ++n;
    }
  } else if (warp == 6) {
    if (p.scale_source != kScalesBulk) {
      Ring<S::kStages> ring;
      int it = 0;
      bool ok = true;
      for (int id = first_item; ok && have; have = next_tile(id)) {
        if (t.expert == p.groups.experts) continue;
        ScaleWords<FMT> ahead[2];  // loads in flight
#pragma unroll
        for (int j = 0; j < 2; ++j) ahead[j] = load_scale_words<FMT>(p, t, min(from + j, to - 1), lane);
        for (int i = from; i < to; ++i, ++it, ring.next()) {
          const ScaleWords<FMT> now = ahead[0];
          ahead[0] = ahead[1];
          if (i + 2 < to) ahead[1] = load_scale_words<FMT>(p, t, i + 2, lane);
          ok = it < S::kStages || pm::mbar_wait(&empty[ring.slot], ring.round ^ 1u, pm::kStatusTimeoutLoad);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          uint8_t* at = smem + ring.slot * S::kStage + S::kW + S::kX + lane * 16;
#pragma unroll
          for (int k = 0; k < S::kTiles; ++k)
            *reinterpret_cast<uint4*>(at + k * 512) = make_uint4(now.w[0][k], now.w[1][k], now.w[2][k], now.w[3][k]);
          pm::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) pm::mbar_arrive(&full[ring.slot]);
        }
      }
    }
  } else if constexpr (kFused) {
    const bool two = FMT == kNV && p.x_second != nullptr;
    const Second second = second_of(two, two ? *p.x_second : 1.0f);
    Ring<S::kStages> ring;
    int it = 0;
    bool ok = true;
    for (int id = first_item; ok && have; have = next_tile(id)) {
      if (t.expert == p.groups.experts) continue;
      const int mine = warp - S::kFirstQuantWarp;
      int i = from + ((mine - it) & (kQuantWarps - 1));  // every fourth stage is this warp's
      TokenBlock<DT> next = first_tokens;
      if (it > 0 && i < to) next = load_tokens<DT>(p, t, i, 0);
      for (; i < to; i += kQuantWarps) {
        const TokenBlock<DT> now = next;
        if (i + kQuantWarps < to) next = load_tokens<DT>(p, t, i + kQuantWarps, 0);
        ring.at(it + (i - from));
        ok = it + (i - from) < S::kStages || pm::mbar_wait(&empty[ring.slot], ring.round ^ 1u, pm::kStatusTimeoutLoad);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        uint8_t* at = smem + ring.slot * S::kStage;
        quantize_tokens<DT, FMT>(p, t, now, i, 0, at + S::kW, at + S::kW + S::kX + S::kSW, second);
        for (int r0 = 2; r0 < t.count; r0 += 2)
          quantize_tokens<DT, FMT>(p, t, load_tokens<DT>(p, t, i, r0), i, r0, at + S::kW, at + S::kW + S::kX + S::kSW, second);
        pm::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) pm::mbar_arrive(&full[ring.slot]);
      }
      it += stages;
    }
  }

  if (S::kCanSplit && p.split > 1) {
    __syncwarp();
    cluster_sync();  // every block's sums are written
    if (find_tile(p.groups, first_item, BN, t) && t.expert != p.groups.experts) {
      float alpha = p.w_second != nullptr ? p.w_second[t.expert] : 1.0f;
      if (p.x_second != nullptr) alpha *= *p.x_second;
      add_cluster_sums<DT>(reinterpret_cast<const float*>(smem), p.y, t, p.rows, alpha, rank, p.split, S::kThreads, p.vec != 0);
    }
    __syncwarp();
    cluster_sync();  // nobody's shared memory goes while others read it
  }
  __syncthreads();
  if (warp == 1) {
    pm::tc_fence_after();
    pm::tmem_dealloc(tmem, S::kAlloc);
  }
}

}  // namespace fp4
