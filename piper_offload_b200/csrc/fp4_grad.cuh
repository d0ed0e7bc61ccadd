// fp4_grad.cuh - dx[t, k] = alpha * sum_n dy[t, n] * w[n, k] with w in packed FP4.
//
// The sum runs over the weight's rows while its scales run along them, so the
// block-scaled instructions do not apply. Instead the weight is decoded on
// chip to bf16, which holds every code times its block scale exactly (at most
// 2 + 4 significant bits), and multiplied on the bf16 tensor pipe with fp32
// sums. A tile is kRows x 128 columns of w (the tensor core's 128-row operand,
// stored with its columns contiguous) x up to BN tokens; a stage is 64 rows of
// w. dy comes by bulk tensor copies; eight warps decode: 16 bytes of codes a
// thread and 128 columns, loaded two stages ahead, looked up by byte permutes,
// scaled by packed bf16 products and written in the 128-byte swizzle.
//
// A stage of 256 columns x 256 tokens keeps the pipe busy for 1024 cycles; the
// pipe reads 96 KB for it and 64 are written, 1280 cycles at 128 bytes each, and
// decoding takes its warps about 900 issue slots of each scheduler, 320 of them
// conversion. A stage takes about 1740 cycles: 2048 x 14336 x 4096 NVFP4 199 us, 1.2
// PFLOP/s (240 in a running program, under the power cap), on 128 of the 148 SMs,
// the pipe active 53 % of the time. Neither side alone bounds it: copies and products
// without the decoding would take 176, decoding with a quarter of the products 174.
// In tiles of 128 columns, whose stages bring 36 KB for 512 cycles, 231. Few tokens:
// decoding, since every value of w is decoded once a tile; 64 x 4096 x 4096 MXFP4
// 14.2 us (cluster of 4, without it 36.5).
//
// fp32 gradients are the sum of three bf16 terms (24 bits): the stages go
// over the weight once per term (2048 x 14336 x 4096 720 to 740 us). The tensor
// core's fp32 additions lose more than rounding to nearest would: over 14336 rows
// 5.5e-6 of the result's norm, against 4.4e-7.
#pragma once
#include <cuda.h>

#include "fp4_ptx.cuh"
#include "fp4_tiles.cuh"

namespace fp4 {

constexpr int kGradStageRows = 64;   // rows of w per stage
constexpr int kDecodeWarps = 8;      // for 64 rows x 128 columns; two such teams a block, which run the epilogue too

struct GradArgs {
  CUtensorMap dy_map;   // (terms * tokens, rows of w) bf16
  const uint8_t* codes;
  const uint8_t* scale;
  const float* second;  // (experts) or NULL
  Groups groups;        // row tiles: of kRows x 128 columns of w
  void* dx;
  int64_t code_pitch;
  int32_t rows, cols;   // of w
  int32_t swizzled;
  int32_t scale_cols;   // scales, or tiles of them, per row
  int32_t terms;
  int32_t split;        // blocks of a cluster that share a tile's stages
  int32_t vec;          // rows of dx start on 16-byte boundaries
  int32_t piece;        // bytes that aligned loads of codes may take: 16, 8 or 1
};

template <int BN, int kRows>
struct GradShape {
  static constexpr int kA = kRows * kGradStageRows * kTileRows * 2;
  static constexpr int kB = BN * kGradStageRows * 2;
  static constexpr int kStage = kA + kB;
  static constexpr int kRoom = kSmemMax - 3072;
  static constexpr int kStages = kRoom / kStage < 8 ? kRoom / kStage : 8;
  static constexpr int kSmem = kStages * kStage + 1024 + 256;
  static constexpr int kThreads = 64 + 32 * kDecodeWarps * 2;  // producer warp, tensor-core warp, decoding warps
  static constexpr int kTurns = 2 / kRows;  // teams that take stages in turn
  static constexpr int kAlloc = kRows * BN;
  static constexpr bool kCanSplit = kRows == 1 && BN * kTileRows * 4 <= kStages * kStage;
  static_assert(kAlloc >= 32 && kAlloc <= 512 && kStages >= 3, "the tile does not fit");
};

// kind::f16, bf16 operands, fp32 sums, A stored M-major (bit 15), B K-major, M = 128.
__device__ __forceinline__ constexpr uint32_t idesc_grad(uint32_t n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// A thread's share of 64 rows x 128 columns: 32 codes of one row and their scales' bytes.
struct Piece {
  uint4 codes;
  uint32_t scale[2];  // MXFP4: both the same
};

// Walks down the weight in stages: this thread's row of each, 32 columns from `col` on.
template <int FMT>
struct PieceWalk {
  const uint8_t* codes;
  const uint8_t* scale;
  int64_t code_step, even_step, odd_step;  // to the next stage; of scales from an even and from an odd one
  int row, rows, bytes, piece, odd;

  __device__ __forceinline__ void begin(const GradArgs& p, int64_t expert, int block, int in_stage, int col) {
    row = block * kGradStageRows + in_stage;
    rows = p.rows;
    bytes = min(16, max((p.cols - col) >> 1, 0));  // 16, 8 at the end of a row, or none
    piece = p.piece;
    odd = block & 1;
    const int at = bytes > 0 ? col : 0;
    const int64_t r = expert * p.rows + row;
    codes = p.codes + r * p.code_pitch + (at >> 1);
    code_step = kGradStageRows * p.code_pitch;
    const int c = at / block_values<FMT>();
    if (p.swizzled) {
      // 64 rows on are two of a tile's four row groups, or the next tile
      scale = p.scale + expert * ((static_cast<int64_t>(p.rows) + 127) >> 7) * p.scale_cols * 512 + swizzled_byte(row, c, p.scale_cols);
      even_step = 8;
      odd_step = static_cast<int64_t>(p.scale_cols) * 512 - 8;
    } else {
      scale = p.scale + r * p.scale_cols + c;
      even_step = odd_step = kGradStageRows * static_cast<int64_t>(p.scale_cols);
    }
  }

  __device__ __forceinline__ Piece load() const {
    Piece out;
    out.codes = make_uint4(0u, 0u, 0u, 0u);
    out.scale[0] = out.scale[1] = 0u;
    if (row >= rows || bytes == 0) return out;
    if (piece == 16 && bytes == 16) {
      out.codes = *reinterpret_cast<const uint4*>(codes);
    } else if (piece >= 8) {
      const uint2 lo = *reinterpret_cast<const uint2*>(codes);
      out.codes.x = lo.x;
      out.codes.y = lo.y;
      if (bytes == 16) {
        const uint2 hi = *reinterpret_cast<const uint2*>(codes + 8);
        out.codes.z = hi.x;
        out.codes.w = hi.y;
      }
    } else {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < bytes) w[i >> 2] |= static_cast<uint32_t>(codes[i]) << (8 * (i & 3));
      out.codes = make_uint4(w[0], w[1], w[2], w[3]);
    }
    out.scale[0] = out.scale[1] = scale[0];
    if (FMT == kNV && bytes == 16) out.scale[1] = scale[1];  // an even block and the next are in one tile
    return out;
  }

  __device__ __forceinline__ void next() {
    codes += code_step;
    scale += odd ? odd_step : even_step;
    odd ^= 1;
    row += kGradStageRows;
  }
};

template <int DT, int FMT, int BN, int kRows>
__global__ void __launch_bounds__(GradShape<BN, kRows>::kThreads, 1) grad_kernel(const __grid_constant__ GradArgs p) {
  using S = GradShape<BN, kRows>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kStages * S::kStage);  // dy landed
  uint64_t* ready = full + S::kStages;                                          // w decoded
  uint64_t* empty = ready + S::kStages;
  uint64_t* done = empty + S::kStages;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == 0 && lane == 0) {
    pm::prefetch_tmap(&p.dy_map);
    for (int s = 0; s < S::kStages; ++s) {
      pm::mbar_init(&full[s], 1);
      pm::mbar_init(&ready[s], kDecodeWarps * kRows);  // of one team, or of both halves'
      pm::mbar_init(&empty[s], 1);
    }
    pm::mbar_init(done, 1);
    pm::fence_mbar_init();
  } else if (warp == 1) {
    pm::tmem_alloc(tmem_at, S::kAlloc);
    pm::tmem_relinquish();
  }
  const int rank = p.split > 1 ? static_cast<int>(cluster_rank()) : 0;
  TileAt t;
  const bool have = find_tile(p.groups, p.split > 1 ? blockIdx.x / p.split : blockIdx.x, BN, t);
  pm::tc_fence_before();
  __syncthreads();
  pm::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_at, 0);
  const int blocks = (p.rows + kGradStageRows - 1) / kGradStageRows;  // of 64 rows of w
  const int all = blocks * p.terms;
  const int from = p.split > 1 ? all * rank / p.split : 0, to = p.split > 1 ? all * (rank + 1) / p.split : all;
  const bool sums = have && t.expert != p.groups.experts;

  if (have && !sums) {
    if (rank == 0)
      for (int h = 0; h < kRows; ++h) {
        TileAt part = t;
        part.row_tile = t.row_tile * kRows + h;
        store_zeros<DT>(p.dx, part, p.cols, threadIdx.x, S::kThreads);
      }
  } else if (sums) {
    if (warp == 0) {
      const int first = __shfl_sync(0xFFFFFFFFu, t.first, 0);
      int issued = 0;
      if (elect_one()) {
        Ring<S::kStages> ring;
        int block = from % blocks, row = first + from / blocks * static_cast<int>(p.groups.tokens);
        for (int i = from; i < to; ++i, ring.next()) {
          if (issued >= S::kStages && !pm::mbar_wait(&empty[ring.slot], ring.round ^ 1u, pm::kStatusTimeoutLoad)) break;
          pm::mbar_arrive_expect_tx(&full[ring.slot], S::kB);
          pm::tma_load_2d(smem + ring.slot * S::kStage + S::kA, &p.dy_map, block * kGradStageRows, row, &full[ring.slot]);
          ++issued;
          if (++block == blocks) {  // the next term
            block = 0;
            row += static_cast<int>(p.groups.tokens);
          }
        }
      }
      __syncwarp();
      issued = __reduce_max_sync(0xFFFFFFFFu, issued);
      // the last copies land before the block's shared memory goes, even if the tensor-core warp gave up
      for (int i = max(0, issued - S::kStages); i < issued; ++i)
        pm::mbar_wait(&full[i % S::kStages], (i / S::kStages) & 1, pm::kStatusTimeoutLoad);
      __syncwarp();
    } else if (warp == 1) {
      const uint32_t idesc = idesc_grad((static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, t.count, 0)) + 15u) & ~15u);
      if (elect_one()) {
        Ring<S::kStages> ring;
        for (int i = from; i < to; ++i, ring.next()) {
          if (!pm::mbar_wait(&full[ring.slot], ring.round, pm::kStatusTimeoutMma) ||
              !pm::mbar_wait(&ready[ring.slot], ring.round, pm::kStatusTimeoutMma))
            break;
          pm::tc_fence_after();
          const uint32_t at = pm::smem_u32(smem) + ring.slot * S::kStage;
          // w: 64-column blocks 8 KB apart, groups of 8 rows 1 KB apart; dy: 128-byte rows of 64 values
          const uint64_t a = pm::smem_desc_sw(at, kGradStageRows * 128, 1024, 2);
          const uint64_t b = pm::smem_desc_sw(at + S::kA, 16, 1024, 2);
#pragma unroll
          for (int j = 0; j < kGradStageRows / 16; ++j)
#pragma unroll
            for (int h = 0; h < kRows; ++h)
              pm::umma_f16(tmem + h * BN, a + h * (kGradStageRows * kTileRows * 2 >> 4) + j * (2048 >> 4), b + j * (32 >> 4), idesc,
                           i != from || j != 0);
          pm::umma_commit(&empty[ring.slot]);
        }
        pm::umma_commit(done);
      }
      __syncwarp();
    } else {
      // a team has 128 columns of every stage, or of every second one: a warp decodes eight rows, a lane 32 columns of
      // one, and the eight lanes whose 16-byte stores go together write different rows, so the swizzle gives them
      // different banks
      const int team = (warp - 2) / kDecodeWarps;
      const int h = kRows == 2 ? team : 0, turn = kRows == 2 ? 0 : team;
      const int r = (warp - 2) % kDecodeWarps * 8 + (lane & 7), quarter = lane >> 3;
      const int col = (t.row_tile * kRows + h) * kTileRows + quarter * 32;
      uint8_t* const to_row = smem + h * (kGradStageRows * kTileRows * 2) + (quarter >> 1) * (kGradStageRows * 128) + r * 128;
      PieceWalk<FMT> walk;
      int block = (from + turn) % blocks;  // of the next loads
      walk.begin(p, t.expert, block, r, col);
      const auto load_next = [&]() {
        const Piece piece = walk.load();
#pragma unroll
        for (int j = 0; j < S::kTurns; ++j) {
          walk.next();
          if (++block == blocks) {  // the next term
            block = 0;
            walk.begin(p, t.expert, 0, r, col);
          }
        }
        return piece;
      };
      Piece soon = load_next(), later = load_next();  // this team's next stage's, the one after's
      Ring<S::kStages> ring;
      if (turn == 1) ring.next();
      bool ok = true;
      for (int i = from + turn; i < to; i += S::kTurns) {
        const Piece now = soon;
        soon = later;
        if (i + 2 * S::kTurns < to) later = load_next();
        if (i - from >= S::kStages) {
          ok = __all_sync(0xFFFFFFFFu, pm::mbar_wait(&empty[ring.slot], ring.round ^ 1u, pm::kStatusTimeoutLoad));
          if (!ok) break;
        }
        uint8_t* row = to_row + ring.slot * S::kStage;
        const uint32_t c[4] = {now.codes.x, now.codes.y, now.codes.z, now.codes.w};
        const __nv_bfloat162 scale[2] = {__float2bfloat162_rn(scale_value<FMT>(now.scale[0])),
                                         __float2bfloat162_rn(scale_value<FMT>(now.scale[1]))};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 v;
          decode4(c[q], scale[q >> 1], v.x, v.y);
          decode4(c[q] >> 16, scale[q >> 1], v.z, v.w);
          *reinterpret_cast<uint4*>(row + ((((quarter & 1) * 4 + q) ^ (r & 7)) << 4)) = v;
        }
        pm::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) pm::mbar_arrive(&ready[ring.slot]);
#pragma unroll
        for (int j = 0; j < S::kTurns; ++j) ring.next();
      }
      ok = __all_sync(0xFFFFFFFFu, pm::mbar_wait(done, 0, pm::kStatusTimeoutMma));
      pm::tc_fence_after();
      if (ok) {
        // the sums are complete, so the stages are free
        if (S::kCanSplit && p.split > 1) {
          if (warp < 6) store_sums(tmem, t, reinterpret_cast<float*>(smem));
        } else {
          const float alpha = p.second != nullptr ? p.second[t.expert] : 1.0f;
          uint8_t* mine = smem + (warp - 2) * 2048;
          TileAt part = t;
          part.row_tile = t.row_tile * kRows + h;
          // 4 / kRows warps for each quarter of the lanes: a share of the tokens each
          constexpr int kShare = BN * kRows / 4 < 32 ? 32 : BN * kRows / 4;
          const int share = (kRows == 2 ? (warp - 2) % kDecodeWarps : warp - 2) / 4;
          store_tile<DT>(tmem + h * BN, p.dx, part, p.cols, alpha, share * kShare, min((share + 1) * kShare, BN), mine, p.vec != 0);
        }
      }
      pm::tc_fence_before();
    }
  }
  if (S::kCanSplit && p.split > 1) {
    __syncwarp();
    cluster_sync();  // every block's sums are written
    if (sums)
      add_cluster_sums<DT>(reinterpret_cast<const float*>(smem), p.dx, t, p.cols, p.second != nullptr ? p.second[t.expert] : 1.0f,
                           rank, p.split, S::kThreads, p.vec != 0);
    __syncwarp();
    cluster_sync();  // nobody's shared memory goes while others read it
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
      // the largest fp32 values round beyond bf16's range: its last number first, and the terms after make up for it
      const float most = __uint_as_float(0x7F7F0000u);
      const __nv_bfloat16 b = __float2bfloat16_rn(isfinite(v) ? fminf(fmaxf(v, -most), most) : v);
      out[i * tokens * pitch + at] = b;
      v = isfinite(v) ? __fsub_rn(v, __bfloat162float(b)) : 0.0f;  // an infinity or a NaN is its first term alone
    }
  }
}

}  // namespace fp4
