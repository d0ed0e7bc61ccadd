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
// A lane holds 16 neighbouring values: one 32-byte load (bf16), one 8-byte
// store, no shuffle for an NVFP4 block and one for an MXFP4 block; four rows are
// in flight per lane, and only a block of threads divides to find its place (8
// values a lane and a division per lane cost twice the time). Bound: HBM for
// fp32 and for dequantising. Codes of bf16 reach neither HBM's rate nor the
// issue slots' (58 % active): rows that wait in registers leave room for four
// blocks an SM, 43 % of the warps, whose first stall is the loads'.
//
// Measured on a B200 (copies run at 6.5 TB/s), one direction again and again:
// 12288 x 3072 bf16 to MXFP4 19.4 us (4.9 TB/s) and back 15.4 (6.2); 4096 x 14336
// to NVFP4, bf16 one level 32 us (4.7), two levels 56, back 25.5 (5.9); fp32 two
// levels 88 us for both passes (5.7), back 43 (6.2).
#pragma once
#include "fp4_ptx.cuh"
#include "numerics.cuh"

namespace fp4 {

enum : int { kMX = 0, kNV = 1 };
enum : int { kBF16 = 0, kF32 = 2 };
enum : int { kFloor = 0, kRceil = 1, kCeil = 2, kEven = 3 };
enum : int { kSecondNone = 0, kSecondGiven = 1, kSecondCompute = 2 };

constexpr int kQuantThreads = 256;
// Rows in flight per lane where there are many (12288 x 3072 bf16 with 4, 2, 1: 23, 26, 31 us; 4096 x 14336 fp32
// two-level: 62, 52, 53), and the blocks per SM that registers leave room for.
template <int DT>
__host__ __device__ constexpr int quant_rows() { return DT == kBF16 ? 4 : 2; }
template <int DT>
constexpr int quant_ctas() { return DT == kBF16 ? 4 : 2; }
constexpr int kDequantRows = 4;
constexpr int kUnit = 16;  // values per lane and row
constexpr int kSmallThreads = 512;

template <int FMT>
__host__ __device__ constexpr int block_values() { return FMT == kMX ? 32 : 16; }
// Columns covered by one 4-scale tile of the swizzled layout.
template <int FMT>
__host__ __device__ constexpr int tile_cols() { return 4 * block_values<FMT>(); }

// Byte of scale (r, c) in the swizzled layout with `ct` tiles per row of tiles.
__host__ __device__ __forceinline__ int64_t swizzled_byte(int64_t r, int c, int ct) {
  const int rin = static_cast<int>(r & 127);
  return ((r >> 7) * ct + (c >> 2)) * 512 + (rin & 31) * 16 + (rin >> 5) * 4 + (c & 3);
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

// Experts of `rows` rows from row0 on: lane j gets row row0 + j's, which is the
// first one whose end is past the row, and the largest end before it (0 without
// one; the ends need not be in order). A warp calls; one load of the ends
// serves all rows (a search by halves a lane took five, 2 us of a 4 us launch).
__device__ __forceinline__ void experts_of_rows(const int32_t* ends, int experts, int64_t row0, int rows, int& expert, int& start) {
  const int lane = threadIdx.x & 31;
  expert = start = 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int32_t v = e0 + lane < experts ? max(ends[e0 + lane], 0) : 0x7FFFFFFF;
    for (int j = 0; j < rows; ++j) {
      // lanes below the first past end
      const uint32_t past = __ballot_sync(0xFFFFFFFFu, v > row0 + j), first = past & (0u - past);
      const int32_t before = __reduce_max_sync(0xFFFFFFFFu, (first - 1u) >> lane & 1u ? v : 0);
      if (lane == j && expert == e0) {
        expert += __popc(first - 1u);
        start = max(start, before);
      }
    }
  }
}

struct QuantArgs {
  const void* x;
  int64_t x_stride;      // values between rows
  int64_t rows;          // rows per matrix
  int64_t rows_padded;   // rows that get scales (a multiple of 128 for swizzled weights)
  int64_t batch;
  int32_t cols;
  int32_t units;         // units of 16 columns per row that are walked (padding included)
  int32_t row_blocks;    // quant_row_blocks of the launch
  int32_t vec;           // rows of x start on 32-byte boundaries
  uint8_t* codes;
  int64_t code_pitch;    // bytes between rows
  uint8_t* scale;
  int32_t scale_cols;    // scales per row (row-major) or tiles per row (swizzled)
  int32_t swizzled;
  int32_t words;         // four scales leave as one aligned word
  int32_t pairs;         // 8-byte stores of codes are aligned
  int32_t pad_codes;     // also write the codes of padding columns (as zeros)
  int32_t scale_mode;
  int32_t second_mode;
  int32_t reverse;       // walk from the end: the maximum pass left that in L2
  float* second;         // (batch): read (given) or written (compute)
  const uint32_t* amax;  // (batch) bits of max|x| over finite values (compute)
  // tokens of experts
  const int32_t* ends;   // NULL: one weight for all
  int32_t experts;
  int32_t token_tile;    // 0: rows are a weight's; else tokens in tiles of so many (first_scale_row)
};

// Lanes that share a row: 32, or fewer (at least a tile of scales) for short rows.
__host__ __device__ __forceinline__ int lanes_per_row(int units) { return units > 16 ? 32 : units > 8 ? 16 : 8; }
// Blocks of kQuantThreads threads that a walk takes: by rows of one matrix, by chunks of 512 columns, in all.
__host__ __device__ __forceinline__ int64_t quant_row_blocks(const QuantArgs& q, int rows_per_lane) {
  const int rows = kQuantThreads / lanes_per_row(q.units) * rows_per_lane;
  return (q.rows_padded + rows - 1) / rows;
}
__host__ __device__ __forceinline__ int quant_chunks(const QuantArgs& q) { return (q.units + 31) / 32; }
__host__ __device__ __forceinline__ int64_t quant_blocks(const QuantArgs& q, int rows_per_lane) {
  return q.batch * quant_row_blocks(q, rows_per_lane) * quant_chunks(q);
}

// 16 neighbouring values as they are stored.
template <int DT>
struct Raw {
  uint32_t w[DT == kBF16 ? 8 : 16];
};

__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

template <int DT>
__device__ __forceinline__ Raw<DT> load_unit(const void* x, int64_t at, bool vec) {
  Raw<DT> r;
  if constexpr (DT == kBF16) {
    const uint16_t* p = static_cast<const uint16_t*>(x) + at;
    if (vec) {
      load32(p, r.w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.w[i] = p[2 * i] | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
    }
  } else {
    const uint32_t* p = static_cast<const uint32_t*>(x) + at;
    if (vec) {
      load32(p, r.w);
      load32(p + 8, r.w + 8);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) r.w[i] = p[i];
    }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void to_floats(const Raw<DT>& r, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if constexpr (DT == kBF16) v[i] = __uint_as_float(i & 1 ? r.w[i >> 1] & 0xFFFF0000u : r.w[i >> 1] << 16);
    else v[i] = __uint_as_float(r.w[i]);
  }
}

__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Bits of max|v|. A NaN stays one, and as an integer it is above infinity.
__device__ __forceinline__ uint32_t amax16(const float (&v)[16]) {
  float m = max3_abs_nan(v[0], v[1], v[2]), n = max3_abs_nan(v[3], v[4], v[5]);
  m = max3_abs_nan(m, v[6], v[7]);
  n = max3_abs_nan(n, v[8], v[9]);
  m = max3_abs_nan(m, v[10], v[11]);
  n = max3_abs_nan(n, v[12], v[13]);
  return __float_as_uint(max3_abs_nan(max3_abs_nan(m, v[14], v[15]), n, n)) & 0x7FFFFFFFu;
}

// a / b rounded to nearest, from r = 1 / b rounded to nearest: Markstein's
// theorem ("Computation of elementary functions on the IBM RISC System/6000
// processor", 1990) makes one residual step exact while nothing under- or
// overflows. For magnitudes within 2^+-60; three instructions.
__device__ __forceinline__ float near_quotient(float a, float b, float r) {
  const float q = __fmul_rn(a, r);
  return __fmaf_rn(__fmaf_rn(-q, b, a), r, q);
}
// Whether a magnitude's bits are those of a number within 2^+-60.
__device__ __forceinline__ bool near_one(uint32_t bits) { return bits - (67u << 23) < (120u << 23); }

__device__ __forceinline__ float sixth(uint32_t amax) {
  const float a = __uint_as_float(amax);
  return near_one(amax) ? near_quotient(a, 6.0f, 1.0f / 6.0f) : __fdiv_rn(a, 6.0f);
}

__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax, int mode) {
  if (amax > 0x7F800000u) return 255u;
  uint32_t bits = amax;
  if (mode == kRceil) bits = __float_as_uint(sixth(amax));
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

// What a lane keeps of a second level for all its blocks.
struct Second {
  float g, inv_g;  // 1 without one
  bool two, near;  // near: g is within 2^+-60
  float inv_mantissa;  // 1 / (1 + (lane % 8) / 8)
};
__device__ __forceinline__ Second second_of(bool two, float g) {
  Second s;
  s.two = two;
  s.g = g;
  s.inv_g = __fdiv_rn(1.0f, g);
  s.near = near_one(__float_as_uint(g));
  s.inv_mantissa = __frcp_rn(1.0f + static_cast<float>(threadIdx.x & 7) * 0.125f);
  return s;
}

__device__ __forceinline__ uint32_t nv_scale_byte(uint32_t amax, const Second& second) {
  float s = sixth(amax);
  if (second.two) s = second.near && near_one(__float_as_uint(s)) ? near_quotient(s, second.g, second.inv_g) : __fdiv_rn(s, second.g);
  if (s != s) return 127u;
  return pm::enc_e4m3(fminf(fmaxf(s, 0.015625f), 448.0f));
}

// 1 / unit rounded to nearest, of the e4m3 number that a byte from 8 to 126
// stands for: the reciprocal of its 4-bit significand, from another lane, with
// the exponent taken off (the whole warp calls).
__device__ __forceinline__ float inverse_unit(uint32_t byte, const Second& second) {
  const float m = __shfl_sync(0xFFFFFFFFu, second.inv_mantissa, byte & 7u);
  return __uint_as_float(__float_as_uint(m) + ((7u - (byte >> 3)) << 23));
}

// Eight values to codes (nearest, ties to even, saturating), the first in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float2* q) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(q[0].x), "f"(q[0].y), "f"(q[1].x), "f"(q[1].y), "f"(q[2].x), "f"(q[2].y), "f"(q[3].x), "f"(q[3].y));
  return w;
}

// Codes of 16 values (the first in the lowest nibble). kQuotient: v / unit is
// wanted, mul = 1 / unit, and one residual step makes v * mul fall on the
// quotient's side of every rounding boundary: boundaries times a 4-bit unit
// are exact in fp32, so a quotient that is not on a boundary is over half an
// ulp away from it, and one that is comes out exactly.
template <bool kQuotient>
__device__ __forceinline__ uint2 encode16(const float (&v)[16], float mul, float unit) {
  float2 q[8];
  const float2 m2 = make_float2(mul, mul), u2 = make_float2(-unit, -unit);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 x = make_float2(v[2 * i], v[2 * i + 1]);
    q[i] = __fmul2_rn(x, m2);
    if constexpr (kQuotient) q[i] = __ffma2_rn(__ffma2_rn(q[i], u2, x), m2, q[i]);
  }
  return make_uint2(e2m1x8(q), e2m1x8(q + 4));
}

struct Coded {
  uint2 codes;
  uint32_t byte;  // the block's scale
};

// One lane's 16 values; an MXFP4 block is two neighbouring lanes (the whole warp calls).
template <int FMT>
__device__ __forceinline__ Coded quantize16(float (&v)[16], int mode, const Second& second) {
  uint32_t m = amax16(v);
  Coded out;
  if constexpr (FMT == kMX) {
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    out.byte = mx_scale_byte(m, mode);
    out.codes = encode16<false>(v, mx_inverse(out.byte), 0.0f);
  } else {
    out.byte = nv_scale_byte(m, second);
    const float unit = pm::dec_e4m3(out.byte), inverse = inverse_unit(out.byte, second);
    if (second.two) {
      const float mul = second.near ? near_quotient(second.inv_g, unit, inverse) : __fdiv_rn(second.inv_g, unit);
      out.codes = encode16<false>(v, mul, 0.0f);
    } else {
      if (m >= 0x7F800000u) {  // keep infinities out of the residual: 2^20 saturates as they do
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = fminf(fmaxf(v[i], -1048576.0f), 1048576.0f);
      }
      out.codes = encode16<true>(v, inverse, unit);
    }
  }
  return out;
}

// The scales of four neighbouring blocks as a word, in the first one's lane.
template <int FMT>
__device__ __forceinline__ uint32_t gather_scales(uint32_t byte) {
  constexpr int kLanes = FMT == kMX ? 2 : 1;
  uint32_t word = byte | (__shfl_down_sync(0xFFFFFFFFu, byte, kLanes) << 8);
  return word | (__shfl_down_sync(0xFFFFFFFFu, word, 2 * kLanes) << 16);
}

// The second-level scale that a finite maximum gives.
__device__ __forceinline__ float second_of_amax(uint32_t amax) {
  return fmaxf(__fdiv_rn(__uint_as_float(amax), 2688.0f), 1.1920928955078125e-07f);
}

// A warp quantizes R rows (more where a row is short) x 512 columns of matrix e.
template <int DT, int FMT, int R>
__device__ __forceinline__ void quantize_rows(const QuantArgs& q, int e, int row0, int chunk, const Second& second) {
  constexpr int kLanes = FMT == kMX ? 2 : 1;  // lanes per block
  const int lane = threadIdx.x & 31, per = lanes_per_row(q.units);
  const int unit = chunk * 32 + (lane & (per - 1));
  const int step = 32 / per;  // rows side by side in the warp
  const int first = row0 + lane / per;
  const bool in_row = unit < q.units, in_cols = unit * kUnit < q.cols;
  // rows that exist, and rows that get scales, from this lane's first on
  const int live = static_cast<int>(q.rows) - first;
  const int kept = in_row ? static_cast<int>(q.rows_padded) - first : 0;
  const int64_t row = e * q.rows + first;

  Raw<DT> raw[R];
  int64_t from = row * q.x_stride + unit * kUnit;
#pragma unroll
  for (int u = 0; u < R; ++u, from += step * q.x_stride) {
    if (in_cols && u * step < live) {
      raw[u] = load_unit<DT>(q.x, from, q.vec != 0);
    } else {
#pragma unroll
      for (auto& w : raw[u].w) w = 0u;
    }
  }
  // where the warp's tokens' scales go, one row a lane, while the values are on their way
  int64_t place = 0;
  if (q.token_tile != 0) {
    const int r = row0 + lane;
    int x = 0, start = 0;
    if (q.ends != nullptr) experts_of_rows(q.ends, q.experts, row0, R * step, x, start);
    if (x >= q.experts || start < 0 || start > r) {
      place = -1;  // a row of no expert
    } else {
      const int o = r - start, tile = o / q.token_tile;
      place = first_scale_row(start, x, q.token_tile) + static_cast<int64_t>(tile) * scale_rows_per_tile(q.token_tile) +
              (o - tile * q.token_tile);
    }
    if (q.ends == nullptr) place = __shfl_sync(0xFFFFFFFFu, place, lane / per);  // this lane's first row's
  }
  // the rows of a warp are aligned to their number, so in the swizzled layout they follow one another by 16 bytes
  const int c = unit / kLanes;
  uint8_t* scale = q.swizzled ? q.scale + e * (q.rows_padded >> 7) * q.scale_cols * 512 +
                                    swizzled_byte(q.token_tile != 0 ? place : first, c, q.scale_cols)
                              : q.scale + row * q.scale_cols + c;
  const int64_t scale_step = q.swizzled ? step * 16 : static_cast<int64_t>(step) * q.scale_cols;
  uint8_t* codes = q.codes + row * q.code_pitch + unit * 8;
#pragma unroll
  for (int u = 0; u < R; ++u, scale += scale_step, codes += step * q.code_pitch) {
    float v[16];
    to_floats(raw[u], v);
    const Coded s = quantize16<FMT>(v, q.scale_mode, second);
    const bool value = u * step < live && in_cols;
    const uint32_t byte = value ? s.byte : 0u;
    const uint32_t word = gather_scales<FMT>(byte);
    uint8_t* at = scale;
    bool keep = u * step < kept;
    if (q.ends != nullptr) {
      const int64_t srow = __shfl_sync(0xFFFFFFFFu, place, u * step + lane / per);
      keep = keep && srow >= 0;
      at = q.scale + swizzled_byte(max(srow, int64_t{0}), c, q.scale_cols);
    }
    if (!keep) continue;
    if (q.words) {
      if (lane % (4 * kLanes) == 0) *reinterpret_cast<uint32_t*>(at) = word;
    } else if (lane % kLanes == 0) {
      *at = static_cast<uint8_t>(byte);
    }
    if (value || (q.pad_codes && u * step < live)) {
      if (q.pairs) {
        *reinterpret_cast<uint2*>(codes) = s.codes;
      } else {
        reinterpret_cast<uint32_t*>(codes)[0] = s.codes.x;
        reinterpret_cast<uint32_t*>(codes)[1] = s.codes.y;
      }
    }
  }
}

// Block `b` of quant_blocks(q).
template <int DT, int FMT, int R>
__device__ __forceinline__ void quantize_block(const QuantArgs& q, uint32_t b) {
  const uint32_t chunks = quant_chunks(q), per = static_cast<uint32_t>(q.row_blocks);
  const uint32_t rb = b / chunks, e = q.batch == 1 ? 0 : rb / per;
  const int chunk = static_cast<int>(b - rb * chunks);
  const int rows = 32 / lanes_per_row(q.units) * R;  // per warp
  const int row0 = static_cast<int>(rb - e * per) * (rows * (kQuantThreads / 32)) + (threadIdx.x >> 5) * rows;
  float g = 1.0f;
  const bool two = FMT == kNV && q.second_mode != kSecondNone;
  if (two) {
    g = q.second_mode == kSecondGiven ? q.second[e] : second_of_amax(q.amax[e]);
    if (q.second_mode == kSecondCompute && rb == e * per && chunk == 0 && threadIdx.x == 0) q.second[e] = g;
  }
  quantize_rows<DT, FMT, R>(q, static_cast<int>(e), row0, chunk, second_of(two, g));
}

template <int DT, int FMT, int R>
__global__ void __launch_bounds__(kQuantThreads, quant_ctas<DT>()) quantize_kernel(const __grid_constant__ QuantArgs q) {
  quantize_block<DT, FMT, R>(q, q.reverse ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// Bits of the largest finite magnitude of a warp's rows x 512 columns, in every
// lane: an infinity or a NaN would take the whole matrix's scale with it.
template <int DT>
__device__ __forceinline__ uint32_t amax_rows(const QuantArgs& q, int64_t e, int64_t row0, int chunk) {
  const int lane = threadIdx.x & 31, per = lanes_per_row(q.units);
  const int unit = chunk * 32 + (lane & (per - 1));
  const int step = 32 / per;
  const int64_t first = row0 + lane / per;
  Raw<DT> raw[quant_rows<DT>()];
#pragma unroll
  for (int u = 0; u < quant_rows<DT>(); ++u) {
    const int64_t r = first + u * step;
    if (unit * kUnit < q.cols && r < q.rows) {
      raw[u] = load_unit<DT>(q.x, (e * q.rows + r) * q.x_stride + unit * kUnit, q.vec != 0);
    } else {
#pragma unroll
      for (auto& w : raw[u].w) w = 0u;
    }
  }
  uint32_t m = 0u;
#pragma unroll
  for (int u = 0; u < quant_rows<DT>(); ++u) {
    float v[16];
    to_floats(raw[u], v);
    m = max(m, amax16(v));
  }
  if (m >= 0x7F800000u) {  // rare: again without them
    m = 0u;
#pragma unroll
    for (int u = 0; u < quant_rows<DT>(); ++u) {
      float v[16];
      to_floats(raw[u], v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t bits = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        m = max(m, bits < 0x7F800000u ? bits : 0u);
      }
    }
  }
  return __reduce_max_sync(0xFFFFFFFFu, m);
}

// max|x| over the finite values of each matrix as integer bits (order does not matter to a maximum).
template <int DT>
__global__ void __launch_bounds__(kQuantThreads) amax_kernel(const __grid_constant__ QuantArgs q, uint32_t* amax) {
  const int chunks = (q.units + 31) / 32, rows = 32 / lanes_per_row(q.units) * quant_rows<DT>();
  const int64_t blocks = quant_row_blocks(q, quant_rows<DT>()) * chunks;
  uint32_t m = 0u;
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int64_t rb = b / chunks;
    m = max(m, amax_rows<DT>(q, blockIdx.y, rb * (rows * (kQuantThreads / 32)) + (threadIdx.x >> 5) * rows,
                             static_cast<int>(b - rb * chunks)));
  }
  __shared__ uint32_t part[kQuantThreads / 32];
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < kQuantThreads / 32; ++i) m = max(m, part[i]);
    atomicMax(amax + blockIdx.y, m);
  }
}

// Both passes over a small matrix in one block, the second from L1: one
// launch instead of a clear, a maximum and a quantisation.
template <int DT, int FMT>
__global__ void __launch_bounds__(kSmallThreads) quantize_small_kernel(const __grid_constant__ QuantArgs q) {
  __shared__ uint32_t part[kSmallThreads / 32];
  const int64_t e = blockIdx.x;
  const int chunks = (q.units + 31) / 32, rows = 32 / lanes_per_row(q.units) * quant_rows<DT>();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pieces = static_cast<int>((q.rows_padded + rows - 1) / rows) * chunks;
  uint32_t m = 0u;
  for (int i = warp; i < pieces; i += kSmallThreads / 32)
    m = max(m, amax_rows<DT>(q, e, static_cast<int64_t>(i / chunks) * rows, i % chunks));
  if (lane == 0) part[warp] = m;
  __syncthreads();
  const float g = second_of_amax(__reduce_max_sync(0xFFFFFFFFu, part[lane % (kSmallThreads / 32)]));
  if (threadIdx.x == 0) q.second[e] = g;
  const Second second = second_of(true, g);
  for (int i = warp; i < pieces; i += kSmallThreads / 32)
    quantize_rows<DT, FMT, quant_rows<DT>()>(q, static_cast<int>(e), i / chunks * rows, i % chunks, second);
}

// ------------------------------------------------------------ back to values
template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return FMT == kMX ? pm::dec_e8m0(byte) : pm::dec_e4m3(byte);
}

// Four codes of `nibbles` (low 16 bits) times a scale, as two bf16 pairs: a
// code times a block scale has at most 6 significant bits, so this is exact.
// The magnitudes' bf16 bytes come from two 8-entry tables; a selector with bit
// 3 set would replicate the byte's sign, which gives the sign bits.
__device__ __forceinline__ void decode4(uint32_t nibbles, __nv_bfloat162 scale, uint32_t& lo, uint32_t& hi) {
  const uint32_t sel = nibbles & 0x7777u;
  const uint32_t top = __byte_perm(0x3F3F3F00u, 0x40404040u, sel);
  const uint32_t low = __byte_perm(0xC0800000u, 0xC0804000u, sel);
  // 0x80 for a positive code, 0xFF for a negative one
  uint32_t sign;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(sign) : "r"(0x80808080u), "r"(nibbles));
  const uint32_t high = top | ((sign << 7) & 0x80808080u);
  uint32_t a = __byte_perm(low, high, 0x5140), b = __byte_perm(low, high, 0x7362);
  __nv_bfloat162 x = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), scale);
  __nv_bfloat162 y = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&b), scale);
  lo = *reinterpret_cast<uint32_t*>(&x);
  hi = *reinterpret_cast<uint32_t*>(&y);
}

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scale;
  const float* second;  // (batch) or NULL
  void* y;
  int64_t rows, batch;
  int32_t cols, swizzled, scale_cols;
  int32_t vec;          // units of codes and of y are aligned
};

// Blocks of threads as in a quantisation without padding.
template <int DT, int FMT>
__global__ void __launch_bounds__(kQuantThreads) dequantize_kernel(const __grid_constant__ DequantArgs d) {
  constexpr int kLanes = FMT == kMX ? 2 : 1;
  const int units = d.cols / kUnit, per = lanes_per_row(units), chunks = (units + 31) / 32, step = 32 / per;
  const int block_rows = kQuantThreads / per * kDequantRows;
  const int64_t row_blocks = (d.rows + block_rows - 1) / block_rows;
  const int64_t rb = blockIdx.x / chunks, e = d.batch == 1 ? 0 : rb / row_blocks;
  const int lane = threadIdx.x & 31;
  const int unit = static_cast<int>(blockIdx.x - rb * chunks) * 32 + (lane & (per - 1));
  const int64_t first = (rb - e * row_blocks) * block_rows + (threadIdx.x >> 5) * (step * kDequantRows) + lane / per;
  const uint8_t* scales = d.swizzled ? d.scale + e * ((d.rows + 127) >> 7) * d.scale_cols * 512 : d.scale + e * d.rows * d.scale_cols;
  const float g = d.second != nullptr ? d.second[e] : 1.0f;
  if (unit >= units) return;
  const int c = unit / kLanes;
  uint2 codes[kDequantRows];
  uint32_t byte[kDequantRows];
#pragma unroll
  for (int u = 0; u < kDequantRows; ++u) {
    const int64_t r = first + u * step;
    codes[u] = make_uint2(0u, 0u);
    byte[u] = 0u;
    if (r < d.rows) {
      byte[u] = d.swizzled ? scales[swizzled_byte(r, c, d.scale_cols)] : scales[r * d.scale_cols + c];
      const uint8_t* from = d.codes + ((e * d.rows + r) * units + unit) * 8;
      if (d.vec) {
        codes[u] = *reinterpret_cast<const uint2*>(from);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          codes[u].x |= static_cast<uint32_t>(from[i]) << (8 * i);
          codes[u].y |= static_cast<uint32_t>(from[4 + i]) << (8 * i);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kDequantRows; ++u) {
    const int64_t r = first + u * step;
    if (r >= d.rows) break;
    const __nv_bfloat162 s = __float2bfloat162_rn(scale_value<FMT>(byte[u]));
    uint32_t w[8];
    decode4(codes[u].x, s, w[0], w[1]);
    decode4(codes[u].x >> 16, s, w[2], w[3]);
    decode4(codes[u].y, s, w[4], w[5]);
    decode4(codes[u].y >> 16, s, w[6], w[7]);
    const int64_t at = ((e * d.rows + r) * units + unit) * kUnit;
    if (DT == kBF16 && d.second == nullptr) {
      // exact as they are
    } else {
      uint32_t f[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[2 * i] = __float_as_uint(__fmul_rn(__uint_as_float(w[i] << 16), g));
        f[2 * i + 1] = __float_as_uint(__fmul_rn(__uint_as_float(w[i] & 0xFFFF0000u), g));
      }
      if constexpr (DT == kBF16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(f[2 * i]), __uint_as_float(f[2 * i + 1]));
          w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
      } else {
        uint32_t* p = static_cast<uint32_t*>(d.y) + at;
        if (d.vec) {
          store32(p, f);
          store32(p + 8, f + 8);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = f[i];
        }
      }
    }
    if constexpr (DT == kBF16) {
      uint16_t* p = static_cast<uint16_t*>(d.y) + at;
      if (d.vec) {
        store32(p, w);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

// The product's copies read codes in rows of whole 16-byte pieces. A weight
// with columns that are no multiple of 32, or that starts elsewhere, is laid
// out so first.
struct RepackArgs {
  const uint8_t* codes;
  uint8_t* codes_out;  // NULL: the codes are used where they are
  int64_t row_bytes;
  int64_t pitch;       // bytes between rows of codes_out (a multiple of 16)
  int64_t pieces;      // 16-byte pieces of codes_out
  int32_t aligned;     // rows start on 8-byte boundaries
};

__device__ __forceinline__ void repack(const RepackArgs& p, int64_t i) {
  if (i >= p.pieces) return;
  const int64_t per = p.pitch >> 4;
  const int64_t row = i / per, at = (i - row * per) * 16;
  const uint8_t* from = p.codes + row * p.row_bytes + at;
  const int bytes = static_cast<int>(min(p.row_bytes - at, int64_t{16}));  // 16 or 8
  uint64_t w[2] = {0u, 0u};
  if (p.aligned) {
    w[0] = *reinterpret_cast<const uint64_t*>(from);
    if (bytes == 16) w[1] = *reinterpret_cast<const uint64_t*>(from + 8);
  } else {
    for (int j = 0; j < bytes; ++j) w[j >> 3] |= static_cast<uint64_t>(from[j]) << (8 * (j & 7));
  }
  *reinterpret_cast<ulonglong2*>(p.codes_out + row * p.pitch + at) = make_ulonglong2(w[0], w[1]);
}

// What a product needs ahead of it, in one launch: blocks below
// `token_blocks` quantize tokens, the others lay codes out.
template <int DT, int FMT, int R>
__global__ void __launch_bounds__(kQuantThreads, quant_ctas<DT>())
    prepare_kernel(const __grid_constant__ QuantArgs q, const __grid_constant__ RepackArgs p, uint32_t token_blocks) {
  grid_launch_dependents();
  if (blockIdx.x < token_blocks) quantize_block<DT, FMT, R>(q, blockIdx.x);
  else repack(p, static_cast<int64_t>(blockIdx.x - token_blocks) * kQuantThreads + threadIdx.x);
}

}  // namespace fp4
