// int8_grad.cuh - dx[t, k] = sum_n dy[t, n] s_w[n] (w[n, k] - z[n]) with w in 8 bits.
//
// The sum runs over the weight's rows, which the scales belong to, so they go into the gradient: a launch before makes
// fp16 values of dy[t, n] s_w[n] (int8_quant.cuh, scale_rows). The weight is decoded on chip to fp16, which holds every
// code less its zero point exactly (nine bits), and multiplied on the fp16 tensor pipe with fp32 sums. A tile is
// kRows x 128 columns of w (the tensor core's 128-row operand, stored with its columns contiguous) x up to BN tokens; a
// stage is 64 rows of w. Gradients come by bulk tensor copies. Sixteen warps decode, in teams that take stages in turn and
// load the codes of their next one before they decode: a byte permute puts each code beside the exponent of 1024, and a
// packed difference takes 1024, the offset and the zero point off.
//
// Decoding is bound by issue: 40 instructions for 32 codes, and what a warp does once a stage (its wait, addresses, fence and
// arrival) as many again. So a thread has 64 codes of a stage: with 32, and every warp in every stage, 2048 rows of 16
// experts of 2048 x 2048 took 35 us instead of 32, 512 rows 33 instead of 26 (36 and 27 since a pair's stages are announced
// over the cluster). Codes that a producer brings to L2 ahead changed neither.
//
// With many tokens shared memory is the bound: for 256 columns x 256 tokens of a stage one SM brings in and reads 176 KB,
// 1375 cycles at 128 bytes, for 1024 cycles of products. So they run on pairs of SMs (kPair): each decodes 2 x 128 of a
// tile's 512 columns and holds half of the tokens, which the tensor cores of both read: 128 KB for the same 1024 cycles.
// The odd block's decoded codes are read by products that a thread of the even block issues, so that thread has to be
// told over the cluster, by one that waits until all before is there. That takes 0.7 us and no decoding warp has it to spare, nor
// one warp for all stages: four take them in turn (1024 x 4096 x 4096 36 us, 38 with three, 57 with one).
// 2048 x 14336 x 4096 takes 190 us with the launch before (31), 1.5 PFLOP/s on the 128 SMs that have a tile; without pairs
// 233 us.
#pragma once
#include <cuda.h>

#include "int8_tiles.cuh"

namespace i8 {

constexpr int kGradStageRows = 64;   // rows of w per stage
constexpr int kDecodeWarps = 16;     // of a block, which run the epilogue too

struct GradArgs {
  CUtensorMap dy_map;   // (terms * tokens, rows of w) fp16
  const uint8_t* codes; // rows start on 16-byte boundaries
  const int8_t* zero;   // or NULL
  const float* back;    // (tokens)
  fp4::Groups groups;   // row tiles: of kRows x 128 columns of w
  void* dx;
  int64_t code_pitch;
  int32_t zero_step;
  int32_t rows, cols;   // of w
  int32_t terms;
  int32_t split;        // blocks of a cluster that share a tile's stages
  int32_t tile_tokens;  // at most BN; of a pair a multiple of 32
  int32_t vec;          // rows of dx start on 16-byte boundaries
};

template <int BN, int kRows, bool kPair>
struct GradShape {
  static constexpr int kA = kRows * kGradStageRows * kTileRows * 2;
  static constexpr int kB = (kPair ? BN / 2 : BN) * kGradStageRows * 2;
  static constexpr int kStage = kA + kB;
  static constexpr int kTokens = BN * 4;
  static constexpr int kRoom = kSmemMax - 3 * 1024 - kTokens;
  static constexpr int kStages = kRoom / kStage < 8 ? kRoom / kStage : 8;
  static constexpr int kSmem = kStages * kStage + kTokens + 1024 + 512;
  // producer warp, tensor-core warp, decoding warps, and of a pair those that announce with the tensor-core warp what is decoded
  static constexpr int kAnnounceWarps = kPair ? 4 : 1;
  static constexpr int kThreads = 64 + 32 * kDecodeWarps + 32 * (kAnnounceWarps - 1);
  static constexpr int kTeams = 4 / kRows;  // of decoding warps, which take stages in turn: 64 codes a thread and stage
  static constexpr int kTeamWarps = kDecodeWarps / kTeams;
  static constexpr int kAlloc = tmem_columns(kRows * BN);
  static constexpr bool kCanSplit = !kPair && kRows == 1 && BN * kTileRows * 4 <= kStages * kStage;
  static_assert(kRows * BN <= kAlloc && kStages >= kTeams, "the tile does not fit");
};

// A thread's share of a stage: 16 codes of every fourth row of four / kRows, of each 128 columns, and the rows' zero points.
template <int kRows>
struct Piece {
  uint4 codes[4 / kRows][kRows];
  int32_t zero[4 / kRows];
};

// Walks down the weight in every kTeams-th stage: this thread's rows of each, at its columns. What lies past the last row or
// column is some other code: gradients are zero there, and columns past the last are not stored.
template <int kRows>
struct PieceWalk {
  static constexpr int kTeams = 4 / kRows;
  const uint8_t* codes;
  const int8_t* zero;
  uint32_t pitch, zero_step, next_columns;  // bytes to the second 128 columns
  int in_stage, last, block, blocks;

  __device__ __forceinline__ void begin(const GradArgs& p, int64_t expert, int row_in_stage, int col, int apart, int first, int all) {
    const int64_t r = expert * p.rows;
    const int64_t at = col < p.code_pitch ? col : 0;  // the pitch is a multiple of 16
    codes = p.codes + r * p.code_pitch + at;
    next_columns = at + apart < p.code_pitch ? apart : 0;
    zero = p.zero != nullptr ? p.zero + r * p.zero_step : nullptr;
    pitch = static_cast<uint32_t>(p.code_pitch);
    zero_step = static_cast<uint32_t>(p.zero_step);
    in_stage = row_in_stage;
    last = p.rows - 1;
    block = first;
    blocks = all;
  }

  __device__ __forceinline__ void load(Piece<kRows>& out) {
#pragma unroll
    for (int q = 0; q < 4 / kRows; ++q) {
      const uint64_t row = static_cast<uint32_t>(min(block * kGradStageRows + in_stage + 4 * q, last));
      const uint8_t* at = codes + row * pitch;
#pragma unroll
      for (int h = 0; h < kRows; ++h) out.codes[q][h] = *reinterpret_cast<const uint4*>(at + (h == 0 ? 0u : next_columns));
      if (zero != nullptr) out.zero[q] = zero[row * zero_step];
    }
    block += kTeams;
    if (block >= blocks) block %= blocks;  // the next term
  }
};

// Four codes, their signs flipped (code + 128), less the zero point, as fp16 in their order. `off`: 1024 + 128 + zero point,
// twice.
__device__ __forceinline__ void decode4(uint32_t u, uint32_t off, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);  // 1024 + code + 128
  const __half2 o = *reinterpret_cast<const __half2*>(&off);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), o), y = __hsub2(*reinterpret_cast<const __half2*>(&b), o);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

// kind::f16 of a pair, M = 256.
__device__ __forceinline__ void umma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int DT, int BN, int kRows, bool kPair>
__global__ void __launch_bounds__(GradShape<BN, kRows, kPair>::kThreads, 1) grad_kernel(const __grid_constant__ GradArgs p) {
  using S = GradShape<BN, kRows, kPair>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  float* token_scale = reinterpret_cast<float*>(smem + S::kStages * S::kStage);
  uint64_t* full = reinterpret_cast<uint64_t*>(token_scale + BN);  // gradients landed (of a pair: both blocks', counted in the even one)
  uint64_t* ready = full + S::kStages;                             // w decoded by this block (in the even one: by both)
  uint64_t* empty = ready + S::kStages;
  uint64_t* done = empty + S::kStages;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t half = kPair ? fp4::cluster_rank() : 0u;  // of a pair
  if (warp == 0 && lane == 0) {
    pm::prefetch_tmap(&p.dy_map);
    for (int s = 0; s < S::kStages; ++s) {
      pm::mbar_init(&full[s], 1);
      pm::mbar_init(&ready[s], S::kTeamWarps + (kPair && half == 0 ? 1 : 0));
      pm::mbar_init(&empty[s], 1);
    }
    pm::mbar_init(done, 1);
    pm::fence_mbar_init();
  } else if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(tmem_at, S::kAlloc);
    } else {
      pm::tmem_alloc(tmem_at, S::kAlloc);
      pm::tmem_relinquish();
    }
  }
  const int rank = !kPair && p.split > 1 ? static_cast<int>(fp4::cluster_rank()) : 0;
  const int sharers = kPair ? 2 : p.split;  // blocks with the same tile
  TileAt t;
  const bool have = fp4::find_tile(p.groups, sharers > 1 ? blockIdx.x / sharers : blockIdx.x, p.tile_tokens, t);
  pm::tc_fence_before();
  __syncthreads();
  fp4::grid_launch_dependents();  // after the allocation (launch.cuh)
  if constexpr (kPair) fp4::cluster_sync();  // both blocks' barriers are there
  pm::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_at, 0);
  const int blocks = (p.rows + kGradStageRows - 1) / kGradStageRows;  // of 64 rows of w
  const int all = blocks * p.terms;
  const int from = p.split > 1 && !kPair ? all * rank / p.split : 0, to = p.split > 1 && !kPair ? all * (rank + 1) / p.split : all;
  const bool sums = have && t.expert != p.groups.experts;
  const RowsOf none{};
  // 128 columns of a tile: the h-th that this block decodes
  const auto column_tile = [&](int h) { return kPair ? (t.row_tile * kRows + h) * 2 + static_cast<int>(half) : t.row_tile * kRows + h; };
  // the tokens that a tile's products take: in sixteens, of a pair in thirty-twos
  constexpr uint32_t kEach = kPair ? 32u : 16u;
  const uint32_t computed = (static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, t.count, 0)) + kEach - 1u) & ~(kEach - 1u);
  fp4::grid_wait();  // gradients, and codes that were laid out, come from the launch before

  if (have && !sums) {
    if (rank == 0)
      for (int h = 0; h < kRows; ++h) {
        TileAt part = t;
        part.row_tile = column_tile(h);
        zero_tile<DT>(p.dx, part, p.cols, threadIdx.x, S::kThreads);
      }
  } else if (sums) {
    if (warp == 0) {
      const int first = __shfl_sync(0xFFFFFFFFu, t.first, 0) + static_cast<int>(half * (computed / 2));
      int issued = 0;
      if (fp4::elect_one()) {
        fp4::Ring<S::kStages> ring;
        int block = from % blocks, row = first + from / blocks * static_cast<int>(p.groups.tokens);
        for (int i = from; i < to; ++i, ring.next()) {
          if (issued >= S::kStages && !mbar_wait_of<kPair>(&empty[ring.slot], ring.round ^ 1u, pm::kStatusTimeoutLoad)) break;
          uint8_t* at = smem + ring.slot * S::kStage + S::kA;
          if constexpr (kPair) {
            if (half == 0) pm::mbar_arrive_expect_tx(&full[ring.slot], 2 * S::kB);
            tma_load_2d_pair(at, &p.dy_map, block * kGradStageRows, row, in_block(pm::smem_u32(&full[ring.slot]), 0));
          } else {
            pm::mbar_arrive_expect_tx(&full[ring.slot], S::kB);
            pm::tma_load_2d(at, &p.dy_map, block * kGradStageRows, row, &full[ring.slot]);
          }
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
      if (half == 0)
        for (int i = max(0, issued - S::kStages); i < issued; ++i)
          mbar_wait_of<kPair>(&full[i % S::kStages], (i / S::kStages) & 1, pm::kStatusTimeoutLoad);
      __syncwarp();
    } else if (warp == 1) {
      const uint32_t idesc = idesc_grad(computed, kPair ? 256u : 128u);
      if (half == 0 && fp4::elect_one()) {
        fp4::Ring<S::kStages> ring;
        for (int i = from; i < to; ++i, ring.next()) {
          if (!mbar_wait_of<kPair>(&full[ring.slot], ring.round, pm::kStatusTimeoutMma) ||
              !mbar_wait_of<kPair>(&ready[ring.slot], ring.round, pm::kStatusTimeoutMma))
            break;
          pm::tc_fence_after();
          const uint32_t at = pm::smem_u32(smem) + ring.slot * S::kStage;
          // w: 64-column blocks 8 KB apart, groups of 8 rows 1 KB apart; gradients: 128-byte rows of 64 values
          const uint64_t a = pm::smem_desc_sw(at, kGradStageRows * 128, 1024, 2);
          const uint64_t b = pm::smem_desc_sw(at + S::kA, 16, 1024, 2);
#pragma unroll
          for (int j = 0; j < kGradStageRows / 16; ++j)
#pragma unroll
            for (int h = 0; h < kRows; ++h) {
              const uint64_t ah = a + h * (kGradStageRows * kTileRows * 2 >> 4) + j * (2048 >> 4), bj = b + j * (32 >> 4);
              if constexpr (kPair) umma_f16_pair(tmem + h * BN, ah, bj, idesc, i != from || j != 0);
              else pm::umma_f16(tmem + h * BN, ah, bj, idesc, i != from || j != 0);
            }
          if constexpr (kPair) umma_commit_pair(&empty[ring.slot]);
          else pm::umma_commit(&empty[ring.slot]);
        }
        if constexpr (kPair) umma_commit_pair(done);
        else pm::umma_commit(done);
      }
      __syncwarp();
    }
    if (kPair && half != 0 && (warp == 1 || warp >= 2 + kDecodeWarps)) {
      // the odd block's stages are announced to the even one, whose thread issues the products for both
      if (fp4::elect_one()) {
        const int first = warp == 1 ? 0 : warp - 1 - kDecodeWarps;
        for (int i = first; i < to - from; i += S::kAnnounceWarps) {
          const int slot = i % S::kStages;
          if (!pm::mbar_wait(&ready[slot], (i / S::kStages) & 1, pm::kStatusTimeoutMma)) break;
          mbar_arrive_pair(in_block(pm::smem_u32(&ready[slot]), 0));
        }
      }
      __syncwarp();
    } else if (warp >= 2 && warp < 2 + kDecodeWarps) {
      // Eight lanes have 64 columns of two rows: of a row's eight 16-byte pieces, XORed with the row, four lanes write the
      // even ones while the four of the row below write the odd ones, to all banks at once.
      const int turn = (warp - 2) / S::kTeamWarps;
      const int r = (warp - 2) % S::kTeamWarps * (16 / kRows) + (lane >> 4) * 2 + (lane >> 2 & 1), right = lane >> 3 & 1, chunk = lane & 3;
      const int at = right * (kGradStageRows * 128) + r * 128 + ((chunk * 2 ^ (r & 7)) << 4);
      const int places[4] = {at, at ^ 16, at ^ 64, at ^ 80};  // of both halves of 16 codes, in rows r + 8 n; in rows r + 4 + 8 n
      if (const int i = threadIdx.x - 64; i < BN) token_scale[i] = i < t.count ? p.back[t.first + i] : 0.0f;
      PieceWalk<kRows> walk;
      walk.begin(p, t.expert, r, column_tile(0) * kTileRows + right * 64 + chunk * 16, kPair ? 2 * kTileRows : kTileRows,
                 (from + turn) % blocks, blocks);
      Piece<kRows> piece;
      walk.load(piece);
      const bool zeros = p.zero != nullptr;
      int slot = turn;
      uint32_t round = 0;
      bool ok = true;
      for (int i = from + turn; i < to; i += S::kTeams) {
        uint32_t u[4 / kRows][kRows][4], off[4 / kRows];
#pragma unroll
        for (int q = 0; q < 4 / kRows; ++q) {
#pragma unroll
          for (int h = 0; h < kRows; ++h) {
            u[q][h][0] = piece.codes[q][h].x ^ 0x80808080u;
            u[q][h][1] = piece.codes[q][h].y ^ 0x80808080u;
            u[q][h][2] = piece.codes[q][h].z ^ 0x80808080u;
            u[q][h][3] = piece.codes[q][h].w ^ 0x80808080u;
          }
          off[q] = 0x64806480u + (zeros ? static_cast<uint32_t>(piece.zero[q]) * 0x10001u : 0u);  // fp16's whole numbers from 1024 on
        }
        if (i + S::kTeams < to) walk.load(piece);
        if (i - from >= S::kStages) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait_of<kPair>(&empty[slot], round ^ 1u, pm::kStatusTimeoutLoad));
          if (!ok) break;
        }
        uint8_t* const stage = smem + slot * S::kStage;
#pragma unroll
        for (int q = 0; q < 4 / kRows; ++q)
#pragma unroll
          for (int h = 0; h < kRows; ++h) {
            uint4 lo, hi;
            decode4(u[q][h][0], off[q], lo.x, lo.y);
            decode4(u[q][h][1], off[q], lo.z, lo.w);
            decode4(u[q][h][2], off[q], hi.x, hi.y);
            decode4(u[q][h][3], off[q], hi.z, hi.w);
            uint8_t* const to_piece = stage + h * (kGradStageRows * kTileRows * 2) + q * 512;
            *reinterpret_cast<uint4*>(to_piece + places[2 * (q & 1)]) = lo;
            *reinterpret_cast<uint4*>(to_piece + places[2 * (q & 1) + 1]) = hi;
          }
        pm::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) pm::mbar_arrive(&ready[slot]);
        if ((slot += S::kTeams) >= S::kStages) {
          slot -= S::kStages;
          round ^= 1u;
        }
      }
      pm::named_bar_sync(1, 32 * kDecodeWarps);  // the tokens' scales are written
      ok = __all_sync(0xFFFFFFFFu, mbar_wait_of<kPair>(done, 0, pm::kStatusTimeoutMma));
      pm::tc_fence_after();
      if (ok) {
        // the sums are complete, so the stages are free
        if (S::kCanSplit && p.split > 1) {
          if (warp < 6) fp4::store_sums(tmem, t, reinterpret_cast<float*>(smem));
        } else {
          uint8_t* mine = smem + (warp - 2) * 2048;
          const int h = kRows == 2 ? (warp - 2) / 8 : 0;
          TileAt part = t;
          part.row_tile = column_tile(h);
          // 4 / kRows warps for each quarter of the lanes: a share of the tokens each
          constexpr int kShare = BN * kRows / 4 < 32 ? 32 : BN * kRows / 4;
          const int share = (kRows == 2 ? (warp - 2) % 8 : warp - 2) / 4;
          store_tile<DT, false>(tmem + h * BN, p.dx, part, p.cols, none, 0, token_scale, nullptr, share * kShare,
                                min((share + 1) * kShare, BN), mine, p.vec != 0);
        }
      }
      pm::tc_fence_before();
    }
  }
  if (S::kCanSplit && p.split > 1) {
    __syncwarp();
    fp4::cluster_sync();  // every block's sums are written
    if (sums)
      add_cluster_sums<DT, false>(reinterpret_cast<const float*>(smem), p.dx, t, p.cols, none, 0, token_scale, nullptr, rank, p.split,
                                  S::kThreads, p.vec != 0);
    __syncwarp();
    fp4::cluster_sync();  // nobody's shared memory goes while others read it
  }
  __syncthreads();
  if constexpr (kPair) fp4::cluster_sync();  // nobody's shared or tensor memory goes while the other block uses it
  if (warp == 1) {
    pm::tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair(tmem, S::kAlloc);
    else pm::tmem_dealloc(tmem, S::kAlloc);
  }
}

}  // namespace i8
