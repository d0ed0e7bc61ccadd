// fp4_quant.cuh - dense <-> packed FP4 conversion kernels.
//
// A block of a row (32 values in MXFP4, 16 in NVFP4) is stored as e2m1 codes
// times one scale. With a = max|x| over the block:
//   MXFP4  scale 2^(e - 127), e from the exponent of a (scale_mode);
//   NVFP4  scale u = e4m3(clamp(a / 6 [/ g], 2^-6, 448)), g the second level;
//   code = e2m1(x / scale), nearest, ties to even, saturating at 6; with a
//   second level x * ((1 / g) / u), each step rounded to fp32.
// These are the merges' formulas (numerics.cuh), with IEEE quotients, and one
// rule of its own: a NaN in a block makes its scale NaN (e8m0 255, e4m3 127),
// so the whole block and what is computed from it read as NaN.
//
// Bound: HBM. One pass, 8 values a lane, so that a warp's loads are whole
// 512-byte (bf16) runs and its code stores 128-byte ones; a block's maximum
// takes one or two shuffles; four scales leave as one word.
#pragma once
#include "fp4_ptx.cuh"
#include "numerics.cuh"

namespace fp4 {

enum : int { kMX = 0, kNV = 1 };
enum : int { kBF16 = 0, kF32 = 2 };
enum : int { kFloor = 0, kRceil = 1, kCeil = 2, kEven = 3 };
enum : int { kSecondNone = 0, kSecondGiven = 1, kSecondCompute = 2 };

constexpr int kQuantThreads = 256;
constexpr int kQuantUnroll = 4;  // octets of 8 values per thread
constexpr int kOctetsPerBlock = kQuantThreads * kQuantUnroll;

template <int FMT>
__host__ __device__ constexpr int block_values() { return FMT == kMX ? 32 : 16; }
// Columns covered by one 4-scale tile of the swizzled layout.
template <int FMT>
__host__ __device__ constexpr int tile_cols() { return 4 * block_values<FMT>(); }

// Byte of scale (r, c) in the swizzled layout with `ct` tiles per row of tiles.
__host__ __device__ __forceinline__ int64_t swizzled_byte(int64_t r, int64_t c, int64_t ct) {
  const int rin = static_cast<int>(r & 127);
  return ((r >> 7) * ct + (c >> 2)) * 512 + (rin & 31) * 16 + (rin >> 5) * 4 + static_cast<int>(c & 3);
}

// Scale rows of tokens. Every tile of `tile` tokens of an expert starts on a
// 128-row tile of scales, because the tensor core reads them from its first
// column. Expert e's first tile is number start / tile + e: with ceil(n / tile)
// tiles of n rows, at least that many numbers lie before it, so no scan over
// the experts is needed.
__host__ __device__ __forceinline__ int scale_rows_per_tile(int tile) { return (tile + 127) & ~127; }
__host__ __device__ __forceinline__ int64_t first_scale_row(int64_t start, int64_t e, int tile) {
  return (start / tile + e) * scale_rows_per_tile(tile);
}

// Expert whose rows hold row t (the first with ends[e] > t, or `experts`).
__device__ __forceinline__ int expert_of_row(const int32_t* ends, int experts, int64_t t) {
  int lo = 0, hi = experts;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

struct QuantArgs {
  const void* x;
  int64_t x_stride;      // values between rows
  int64_t rows;          // rows per matrix
  int64_t rows_padded;   // rows that get scales (a multiple of 128 when swizzled, without `ends`)
  int64_t batch;
  int32_t cols;
  int32_t octets;        // octets per row that are walked (padding included)
  int32_t vec;           // rows of x start on 16-byte boundaries
  uint8_t* codes;
  int64_t code_pitch;    // bytes between rows
  uint8_t* scale;
  int32_t scale_cols;    // scales per row (row-major) or tiles per row (swizzled)
  int32_t swizzled;
  int32_t words;         // four scales leave as one word: lanes and words stay aligned across rows
  int32_t pad_codes;     // also write the codes of padding columns (as zeros)
  int32_t scale_mode;
  int32_t second_mode;
  int32_t reverse;       // walk from the end: the maximum pass left that in L2
  float* second;         // (batch): read (given) or written (compute)
  const uint32_t* amax;  // (batch) bits of max|x| (compute)
  // tokens of experts
  const int32_t* ends;   // NULL: one weight for all
  int32_t experts;
  int32_t token_tile;    // 0: rows are a weight's; else tokens in tiles of so many (first_scale_row)
};

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t at, bool vec, float (&v)[8]) {
  if constexpr (DT == kBF16) {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if (vec) {
      const uint4 q = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(static_cast<uint32_t>(p[i]) << 16);
    }
  } else {
    const float* p = static_cast<const float*>(base) + at;
    if (vec) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
  }
}

// Bits of max|v|: as integers a NaN is above infinity, so it is never lost.
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax, int mode) {
  if (amax > 0x7F800000u) return 255u;
  uint32_t bits = amax;
  if (mode == kRceil) bits = __float_as_uint(__fdiv_rn(__uint_as_float(amax), 6.0f));
  else if (mode == kEven) bits += 1u << 21;
  int e = static_cast<int>(bits >> 23);
  // above a power of two; 2^-127, the least scale, is half the least normal number
  if ((mode == kRceil || mode == kCeil) && (bits & 0x7FFFFFu) > (e == 0 ? 1u << 22 : 0u)) ++e;
  if (mode != kRceil) e -= 2;
  return static_cast<uint32_t>(min(max(e, 0), 254));
}

// 2^(127 - byte), exact for every finite scale.
__device__ __forceinline__ float mx_inverse(uint32_t byte) {
  return __uint_as_float(byte >= 254u ? (1u << 22) : (254u - byte) << 23);
}

__device__ __forceinline__ uint32_t nv_scale_byte(uint32_t amax, bool two, float g) {
  float s = __fdiv_rn(__uint_as_float(amax), 6.0f);
  if (two) s = __fdiv_rn(s, g);
  if (s != s) return 127u;
  return pm::enc_e4m3(fminf(fmaxf(s, 0.015625f), 448.0f));
}

// Codes of 8 values (the first in the lowest nibble). `mul` multiplies; where
// `unit` is nonzero the quotient v / unit is wanted instead and mul = 1 / unit:
// one residual step makes v * mul the correctly rounded quotient's side of
// every rounding boundary (boundaries times a 4-bit unit are exact in fp32, so
// a quotient that is not on a boundary is over half an ulp away from it, and
// one that is comes out exactly).
__device__ __forceinline__ uint32_t encode8(const float (&v)[8], float mul, float unit) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = __fmul_rn(v[i], mul);
    if (unit != 0.0f) q[i] = __fmaf_rn(__fmaf_rn(-q[i], unit, v[i]), mul, q[i]);
  }
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= pm::enc_e2m1x2(q[2 * i], q[2 * i + 1]) << (8 * i);
  return w;
}

template <int FMT>
struct Scaled {
  uint32_t byte, codes;
};

// One lane's 8 values of a block that spans neighbouring lanes (all of which call).
template <int FMT>
__device__ __forceinline__ Scaled<FMT> quantize8(float (&v)[8], int mode, bool two, float g, float inv_g) {
  uint32_t m = amax8(v);
  m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
  if constexpr (FMT == kMX) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
  Scaled<FMT> out;
  if constexpr (FMT == kMX) {
    out.byte = mx_scale_byte(m, mode);
    out.codes = encode8(v, mx_inverse(out.byte), 0.0f);
  } else {
    out.byte = nv_scale_byte(m, two, g);
    const float unit = pm::dec_e4m3(out.byte);
    if (two) {
      out.codes = encode8(v, __fdiv_rn(inv_g, unit), 0.0f);
    } else {
      if (m >= 0x7F800000u) {  // keep infinities out of the residual: 2^20 saturates as they do
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fminf(fmaxf(v[i], -1048576.0f), 1048576.0f);
      }
      out.codes = encode8(v, __fdiv_rn(1.0f, unit), unit);
    }
  }
  return out;
}

// A whole block of threads quantizes the octets [first, first + kOctetsPerBlock)
// of a walk over batch x rows_padded x octets.
template <int DT, int FMT>
__device__ void quantize_octets(const QuantArgs& q, int64_t first) {
  constexpr int kLanes = FMT == kMX ? 4 : 2;  // lanes per block
  const int64_t total = q.batch * q.rows_padded * q.octets;
  const int64_t row0 = first / q.octets;
  const uint32_t col0 = static_cast<uint32_t>(first - row0 * q.octets);
  const bool words = q.words != 0;
  const uint32_t lane = threadIdx.x & 31u;

  float v[kQuantUnroll][8];
  int64_t row[kQuantUnroll];
  uint32_t oct[kQuantUnroll];
  bool inside[kQuantUnroll];
#pragma unroll
  for (int u = 0; u < kQuantUnroll; ++u) {
    const uint32_t k = col0 + u * kQuantThreads + threadIdx.x;
    const uint32_t r = k / static_cast<uint32_t>(q.octets);
    row[u] = row0 + r;
    oct[u] = k - r * q.octets;
    inside[u] = first + u * kQuantThreads + threadIdx.x < total;
    const int64_t e = q.batch == 1 ? 0 : row[u] / q.rows_padded;
    const int64_t rin = row[u] - e * q.rows_padded;
    if (inside[u] && rin < q.rows && static_cast<int>(oct[u]) * 8 < q.cols) {
      load8<DT>(q.x, (e * q.rows + rin) * q.x_stride + oct[u] * 8, q.vec != 0, v[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < kQuantUnroll; ++u) {
    const int64_t e = q.batch == 1 ? 0 : row[u] / q.rows_padded;
    const int64_t rin = row[u] - e * q.rows_padded;
    float g = 1.0f, inv_g = 1.0f;
    const bool two = FMT == kNV && q.second_mode != kSecondNone;
    if (two && inside[u]) {
      if (q.second_mode == kSecondGiven) {
        g = q.second[e];
      } else {
        // not fmaxf: a NaN maximum stays one
        g = __fdiv_rn(__uint_as_float(q.amax[e]), 2688.0f);
        if (g < 1.1920928955078125e-07f) g = 1.1920928955078125e-07f;
        if (rin == 0 && oct[u] == 0) q.second[e] = g;
      }
      inv_g = __fdiv_rn(1.0f, g);
    }
    const Scaled<FMT> s = quantize8<FMT>(v[u], q.scale_mode, two, g, inv_g);
    const bool live = rin < q.rows;
    const bool padding = !live || static_cast<int>(oct[u]) * 8 >= q.cols;
    const uint32_t byte = padding ? 0u : s.byte;
    // gather the scales of this lane and the next three blocks
    uint32_t word = byte;
    word |= __shfl_down_sync(0xFFFFFFFFu, word, kLanes) << 8;
    word |= __shfl_down_sync(0xFFFFFFFFu, word, 2 * kLanes) << 16;
    if (!inside[u]) continue;

    int64_t srow = rin;
    if (q.token_tile != 0) {
      int x = 0;
      int64_t start = 0;
      if (q.ends != nullptr) {
        x = expert_of_row(q.ends, q.experts, rin);
        start = x > 0 ? q.ends[x - 1] : 0;
        if (x >= q.experts || start < 0 || start > rin) continue;  // a row of no expert
      }
      const int o = static_cast<int>(rin - start);
      srow = first_scale_row(start, x, q.token_tile) +
             static_cast<int64_t>(o / q.token_tile) * scale_rows_per_tile(q.token_tile) + o % q.token_tile;
    }
    const int c = static_cast<int>(oct[u]) / kLanes;
    const int lanes = static_cast<int>(oct[u]) % kLanes;
    if (q.swizzled) {
      uint8_t* base = q.scale + (e * (q.rows_padded >> 7)) * static_cast<int64_t>(q.scale_cols) * 512;
      uint8_t* at = base + swizzled_byte(srow, c, q.scale_cols);
      if (words) {
        if (lane % (4 * kLanes) == 0) *reinterpret_cast<uint32_t*>(at) = word;
      } else if (lanes == 0) {
        *at = static_cast<uint8_t>(byte);
      }
    } else {
      uint8_t* at = q.scale + (e * q.rows + rin) * q.scale_cols + c;
      if (words) {
        if (lane % (4 * kLanes) == 0) *reinterpret_cast<uint32_t*>(at) = word;
      } else if (lanes == 0) {
        *at = static_cast<uint8_t>(byte);
      }
    }
    if (live && (q.pad_codes || !padding))
      *reinterpret_cast<uint32_t*>(q.codes + (e * q.rows + rin) * q.code_pitch + oct[u] * 4) = s.codes;
  }
}

template <int DT, int FMT>
__global__ void __launch_bounds__(kQuantThreads) quantize_kernel(const __grid_constant__ QuantArgs q) {
  const int64_t b = q.reverse ? gridDim.x - 1 - static_cast<int64_t>(blockIdx.x) : blockIdx.x;
  quantize_octets<DT, FMT>(q, b * kOctetsPerBlock);
}

// max|x| of each matrix as integer bits (order does not matter to a maximum).
template <int DT>
__global__ void __launch_bounds__(kQuantThreads) amax_kernel(const __grid_constant__ QuantArgs q, uint32_t* amax) {
  const int64_t octets = q.cols / 8;
  const int64_t total = q.rows * octets;
  const int64_t e = blockIdx.y;
  uint32_t m = 0u;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kOctetsPerBlock;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kOctetsPerBlock; first < total; first += step) {
    const int64_t row0 = first / octets;
    const uint32_t col0 = static_cast<uint32_t>(first - row0 * octets);
    float v[kQuantUnroll][8];
#pragma unroll
    for (int u = 0; u < kQuantUnroll; ++u) {
      const uint32_t k = col0 + u * kQuantThreads + threadIdx.x;
      const uint32_t r = k / static_cast<uint32_t>(octets);
      if (first + u * kQuantThreads + threadIdx.x < total) {
        load8<DT>(q.x, (e * q.rows + row0 + r) * q.x_stride + (k - r * octets) * 8, q.vec != 0, v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < kQuantUnroll; ++u) m = max(m, amax8(v[u]));
  }
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  __shared__ uint32_t part[kQuantThreads / 32];
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < kQuantThreads / 32; ++i) m = max(m, part[i]);
    atomicMax(amax + e, m);
  }
}

// ------------------------------------------------------------ back to values
struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scale;
  const float* second;  // (batch) or NULL
  void* y;
  int64_t rows, batch;
  int32_t cols, swizzled, scale_cols, vec;  // vec: codes and y allow whole-octet accesses
};

template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return FMT == kMX ? pm::dec_e8m0(byte) : pm::dec_e4m3(byte);
}

template <int DT, int FMT>
__global__ void __launch_bounds__(kQuantThreads) dequantize_kernel(const __grid_constant__ DequantArgs d) {
  constexpr int kLanes = FMT == kMX ? 4 : 2;
  const int64_t octets = d.cols / 8;
  const int64_t total = d.batch * d.rows * octets;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kOctetsPerBlock;
  const int64_t row0 = first / octets;
  const uint32_t col0 = static_cast<uint32_t>(first - row0 * octets);
  const int64_t rt = (d.rows + 127) >> 7;
#pragma unroll
  for (int u = 0; u < kQuantUnroll; ++u) {
    const uint32_t k = col0 + u * kQuantThreads + threadIdx.x;
    const uint32_t r = k / static_cast<uint32_t>(octets);
    const int64_t row = row0 + r;
    const uint32_t oct = k - r * static_cast<uint32_t>(octets);
    if (first + u * kQuantThreads + threadIdx.x >= total) break;
    const int64_t e = d.batch == 1 ? 0 : row / d.rows;
    const int c = static_cast<int>(oct) / kLanes;
    const uint8_t* sp = d.swizzled ? d.scale + e * rt * d.scale_cols * 512 + swizzled_byte(row - e * d.rows, c, d.scale_cols)
                                   : d.scale + row * d.scale_cols + c;
    const float s = scale_value<FMT>(*sp);
    const float g = d.second != nullptr ? d.second[e] : 1.0f;
    const uint8_t* cp = d.codes + (row * octets + oct) * 4;
    uint32_t w;
    if (d.vec) {
      w = *reinterpret_cast<const uint32_t*>(cp);
    } else {
      w = cp[0] | (cp[1] << 8) | (cp[2] << 16) | (static_cast<uint32_t>(cp[3]) << 24);
    }
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pm::dec_e2m1x2((w >> (8 * i)) & 0xFFu, v[2 * i], v[2 * i + 1]);
      v[2 * i] = __fmul_rn(__fmul_rn(v[2 * i], s), g);
      v[2 * i + 1] = __fmul_rn(__fmul_rn(v[2 * i + 1], s), g);
    }
    const int64_t at = (row * octets + oct) * 8;
    if constexpr (DT == kBF16) {
      uint16_t* p = static_cast<uint16_t*>(d.y) + at;
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        o[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
      if (d.vec) {
        *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[2 * i] = static_cast<uint16_t>(o[i]);
          p[2 * i + 1] = static_cast<uint16_t>(o[i] >> 16);
        }
      }
    } else {
      float* p = static_cast<float*>(d.y) + at;
      if (d.vec) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = v[i];
      }
    }
  }
}

// ------------------------------------------- weights in the product's layout
// The product reads codes in rows of whole 16-byte pieces and scales in the
// swizzled layout with zeroed padding. Weights stored otherwise are laid out
// by this kernel first: row-major scales, columns that are no multiple of 64
// (padding inside a tile that is used), or unaligned buffers.
struct RepackArgs {
  const uint8_t* codes;
  uint8_t* codes_out;   // NULL: the codes are used where they are
  int64_t code_row;     // bytes of a row
  int64_t code_pitch;   // bytes between rows of codes_out (a multiple of 16)
  const uint8_t* scale;
  uint8_t* scale_out;   // NULL: the scales are used where they are
  int64_t rows, batch;
  int32_t scale_cols;   // scales per row
  int32_t swizzled;     // layout of `scale`
  int64_t words;        // 4-byte words of scale_out
  int64_t pieces;       // 16-byte pieces of codes_out
};

__device__ __forceinline__ void repack(const RepackArgs& p, int64_t i) {
  const int64_t ct = (p.scale_cols + 3) >> 2, rt = (p.rows + 127) >> 7;
  if (i < p.words) {
    const int grp = static_cast<int>(i & 3), lane = static_cast<int>((i >> 2) & 31);
    const int64_t tile = i >> 7;
    const int64_t tc = tile % ct, tr = (tile / ct) % rt, e = tile / (ct * rt);
    const int64_t row = tr * 128 + grp * 32 + lane;
    uint32_t w = 0u;
    if (row < p.rows) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t c = tc * 4 + j;
        if (c < p.scale_cols) {
          const uint8_t* s = p.swizzled ? p.scale + e * rt * ct * 512 + swizzled_byte(row, c, ct)
                                        : p.scale + (e * p.rows + row) * p.scale_cols + c;
          w |= static_cast<uint32_t>(*s) << (8 * j);
        }
      }
    }
    reinterpret_cast<uint32_t*>(p.scale_out)[i] = w;
    return;
  }
  i -= p.words;
  if (i >= p.pieces) return;
  const int64_t per = p.code_pitch >> 4;
  const int64_t row = i / per, at = (i - row * per) * 16;
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (at + j < p.code_row) w[j >> 2] |= static_cast<uint32_t>(p.codes[row * p.code_row + at + j]) << (8 * (j & 3));
  *reinterpret_cast<uint4*>(p.codes_out + row * p.code_pitch + at) = make_uint4(w[0], w[1], w[2], w[3]);
}

// What a product needs ahead of it, in one launch: blocks below
// `quant_blocks` quantize tokens, the others lay weights out.
template <int DT, int FMT>
__global__ void __launch_bounds__(kQuantThreads)
    prepare_kernel(const __grid_constant__ QuantArgs q, const __grid_constant__ RepackArgs p, uint32_t quant_blocks) {
  grid_launch_dependents();
  if (blockIdx.x < quant_blocks) quantize_octets<DT, FMT>(q, static_cast<int64_t>(blockIdx.x) * kOctetsPerBlock);
  else repack(p, static_cast<int64_t>(blockIdx.x - quant_blocks) * kQuantThreads + threadIdx.x);
}

}  // namespace fp4
