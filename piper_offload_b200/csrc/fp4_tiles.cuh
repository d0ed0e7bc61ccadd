// fp4_tiles.cuh - which tile a block works on, shared by the FP4 products and gradients.
#pragma once
#include "fp4_ptx.cuh"
#include "fp4_quant.cuh"

namespace fp4 {

constexpr int kTileRows = 128;  // weight rows (or columns, for a gradient) per tile
constexpr int kSmemMax = 232448;

// Tokens split among experts, and how many row tiles each expert's weight has.
struct Groups {
  const int32_t* ends;  // (experts) or NULL: one weight for all tokens
  int64_t tokens;
  int32_t experts;
  int32_t row_tiles;
};

struct TileAt {
  int32_t expert;        // == experts: rows of no expert, whose results are zero
  int32_t row_tile;
  int32_t first, count;  // token rows of the tile
  int32_t scale_row;     // scale row of the tile's first token (first_scale_row), a multiple of 128
};

// The tile of work item `id`: token tiles are the inner index, so that the
// tiles of one weight strip run together and its bytes are read from HBM once.
// One warp calls; false past the last item. Ends are taken within the tokens,
// and one below an end before it as that end, so that every row has one tile of
// one expert: a vote where they are in order. Few instructions, since every role
// of a block has a copy (a scan by halves cost 24 x 4096 x 4096 MXFP4 0.2 us of 9).
__device__ __forceinline__ bool find_tile(const Groups& p, int id, int bn, TileAt& t) {
  const int tokens = static_cast<int>(p.tokens);
  if (p.ends == nullptr) {
    const int per = (tokens + bn - 1) / bn;
    t.expert = 0;
    t.row_tile = id / per;
    const int nt = id - t.row_tile * per;
    t.first = nt * bn;
    t.scale_row = nt * scale_rows_per_tile(bn);
    t.count = min(bn, tokens - t.first);
    return t.row_tile < p.row_tiles;
  }
  const int lane = threadIdx.x & 31;
  int before = 0;  // tiles of tokens
  int last = 0;  // the end before the first lane's
  for (int e0 = 0; e0 <= p.experts; e0 += 32) {
    const int e = e0 + lane;
    int start, end = e < p.experts ? min(max(p.ends[e], 0), tokens) : tokens;
    for (;; end = max(end, start)) {
      start = __shfl_up_sync(0xFFFFFFFFu, end, 1);
      if (lane == 0) start = last;
      if (!__any_sync(0xFFFFFFFFu, end < start)) break;
    }
    const int n = end - start, per = (n + bn - 1) / bn;
    int sum = per;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, static_cast<int64_t>(before + sum) * p.row_tiles > id);
    if (hit != 0u) {
      const int l = __ffs(hit) - 1;
      const int per_l = __shfl_sync(0xFFFFFFFFu, per, l);
      const int start_l = __shfl_sync(0xFFFFFFFFu, start, l);
      const int n_l = __shfl_sync(0xFFFFFFFFu, n, l);
      const int in = id - (before + __shfl_sync(0xFFFFFFFFu, sum, l) - per_l) * p.row_tiles;
      t.expert = e0 + l;
      t.row_tile = in / per_l;
      const int nt = in - t.row_tile * per_l;
      t.first = start_l + nt * bn;
      t.count = min(bn, n_l - nt * bn);
      t.scale_row = static_cast<int>(first_scale_row(start_l, t.expert, bn)) + nt * scale_rows_per_tile(bn);
      return true;
    }
    before += __shfl_sync(0xFFFFFFFFu, sum, 31);
    last = __shfl_sync(0xFFFFFFFFu, end, 31);
  }
  return false;
}

template <int DT>
__device__ __forceinline__ void store_value(void* y, int64_t at, float v) {
  if constexpr (DT == kBF16) static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else static_cast<float*>(y)[at] = v;
}

// `threads` threads zero a tile of y (tokens x cols).
template <int DT>
__device__ __forceinline__ void store_zeros(void* y, const TileAt& t, int cols, int thread, int threads) {
  const int c0 = t.row_tile * kTileRows, n = min(kTileRows, cols - c0);
  for (int i = thread; i < t.count * kTileRows; i += threads)
    if ((i & (kTileRows - 1)) < n)
      store_value<DT>(y, static_cast<int64_t>(t.first + i / kTileRows) * cols + c0 + (i & (kTileRows - 1)), 0.0f);
}

// Four warps leave a tile's sums in shared memory as (token, 128 outputs).
__device__ __forceinline__ void store_sums(uint32_t tmem, const TileAt& t, float* sums) {
  const int quarter = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  for (int c = 0; c < t.count; c += 32) {
    float v[32];
    pm::tmem_ld32(at + c, v);
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (c + j < t.count) sums[(c + j) * kTileRows + quarter * 32 + lane] = v[j];
  }
}

// A block adds up its share of a tile over the cluster, in rank order: four
// outputs of a token a thread, the ranks' values all in flight at once.
template <int DT>
__device__ __forceinline__ void add_cluster_sums(const float* sums, void* y, const TileAt& t, int cols, float alpha, int rank,
                                                 int split, int threads, bool vec) {
  const uint32_t base = pm::smem_u32(sums);
  const int n0 = t.row_tile * kTileRows;
  for (int i = rank * threads + threadIdx.x; i < t.count * (kTileRows / 4); i += split * threads) {
    const int n = n0 + (i % (kTileRows / 4)) * 4;
    if (n >= cols) continue;
    float4 v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < split) v[r] = load_cluster(base + i * 16, r);
    float4 sum = v[0];
#pragma unroll
    for (int r = 1; r < 8; ++r)
      if (r < split) {
        sum.x += v[r].x;
        sum.y += v[r].y;
        sum.z += v[r].z;
        sum.w += v[r].w;
      }
    sum.x *= alpha;
    sum.y *= alpha;
    sum.z *= alpha;
    sum.w *= alpha;
    const int64_t at = static_cast<int64_t>(t.first + i / (kTileRows / 4)) * cols + n;
    if (vec) {  // rows are 16-byte aligned, so the four outputs exist and lie together
      if constexpr (DT == kBF16) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(y) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else {
        *reinterpret_cast<float4*>(static_cast<float*>(y) + at) = sum;
      }
    } else {
      const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < cols) store_value<DT>(y, at + k, f[k]);
    }
  }
}

// Four epilogue warps' share of a finished tile: tensor-memory lane = column of
// y, tensor-memory column = token, so that a warp's 32 lanes are neighbours in
// y's rows. bf16: 32 tokens at a time are read as the fragments of 8x8
// matrices, rounded, transposed by stmatrix into the warp's own 2 KB of shared
// memory (`stage`; 64-byte rows, 16-byte pieces XORed with the row against
// bank conflicts) and leave as 16-byte pieces of y's rows: 4 stores per 32 x 32
// outputs instead of 32. fp32: a token's 32 outputs are one 128-byte run.
template <int DT>
__device__ __forceinline__ void store_tile(uint32_t tmem, void* y, const TileAt& t, int cols, float alpha, int from_col,
                                           int to_col, uint8_t* stage, bool vec) {
  const int quarter = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const int n0 = t.row_tile * kTileRows + quarter * 32;
  const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const int end = min(to_col, t.count);
  if constexpr (DT == kBF16) {
    const uint32_t base = pm::smem_u32(stage);
    const int piece = lane & 3;
    const int left = cols - n0 - piece * 8;  // outputs of this lane's piece that exist
    for (int c = from_col; c < end; c += 32) {
      uint32_t lo[16], hi[16];
      tmem_ld_fragments(at + c, lo);
      tmem_ld_fragments(at + (16u << 16) + c, hi);
      tmem_ld_fragments_wait(lo, hi);
      __syncwarp();  // the warp has read the last 32 tokens out of its stage
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int token = j * 8 + (lane & 7);
        const uint32_t to = base + token * 64 + (((lane >> 3) ^ ((token >> 1) & 3)) << 4);
        stmatrix_trans(to, bf16_pair(lo[4 * j], lo[4 * j + 1], alpha), bf16_pair(lo[4 * j + 2], lo[4 * j + 3], alpha),
                       bf16_pair(hi[4 * j], hi[4 * j + 1], alpha), bf16_pair(hi[4 * j + 2], hi[4 * j + 3], alpha));
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
    for (int c = from_col; c < end; c += 32) {
      float v[32];
      pm::tmem_ld32(at + c, v);
      if (n < cols) {
        float* to = static_cast<float*>(y) + (static_cast<int64_t>(t.first + c) * cols + n);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < end) to[static_cast<int64_t>(j) * cols] = v[j] * alpha;
      }
    }
  }
}

}  // namespace fp4
