// int8_quant.cuh - what goes before an INT8 product or gradient: tokens to 8 bits, gradients to scaled fp16, codes to aligned rows.
//
// A token x is held as codes q = rint(127 x / a), nearest with ties to even, a = max|x|, and the scale a / 127. Codes are
// those of the exact quotient: 127 x is exact in fp32 for 16-bit x, the quotient gets one residual step (exact where it is
// representable, so ties fall as they should), and no other quotient of two such numbers comes nearer than 2^-19 of itself
// to half a code, where fp32 has 2^-23. For fp32 tokens the remainder decides where the quotient rounds onto a half.
// A row that holds an infinity or a NaN gets the scale NaN: its products are NaN, and no other row's are touched.
//
// Memory bounds it, less its latency, which the blocks that registers leave room for do not cover: 4096 x 4096 bf16 to codes
// 10.4 us, 4.8 TB/s; 2048 x 14336 bf16 gradients to fp16 30 us, 3.9 TB/s.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "fp4_ptx.cuh"

namespace i8 {

enum : int { kBF16 = 0, kF16 = 1, kF32 = 2 };

// Threads of a block whose rows are worked on by so many warps: a row a warp, or a row a block.
__host__ __device__ constexpr int prepare_threads(int warps) { return warps == 1 ? 256 : 32 * warps; }
constexpr int kUnit = 16;  // values that a lane takes at once

// Sixteen values as they lie in memory.
template <int DT>
struct Unit {
  uint32_t w[DT == kF32 ? 16 : 8];
};

template <int DT>
__device__ __forceinline__ float unit_value(const Unit<DT>& u, int i) {
  if constexpr (DT == kF32) return __uint_as_float(u.w[i]);
  const uint32_t w = u.w[i >> 1];
  if constexpr (DT == kBF16) return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return i & 1 ? __high2float(h) : __low2float(h);
}

// Values [col, col + 16) of the row at `row`; those from `cols` on are zero. kVec: rows start on 16-byte boundaries and have
// whole units, so that a row's loads are all in flight together; with a second form of load beside it they are not.
template <int DT, bool kVec>
__device__ __forceinline__ Unit<DT> load_unit(const void* row, int col, int cols) {
  constexpr int kWords = DT == kF32 ? 16 : 8;
  Unit<DT> u;
  if constexpr (kVec) {
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(row) + static_cast<int64_t>(col) * (DT == kF32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const uint4 q = from[i];
      u.w[4 * i] = q.x; u.w[4 * i + 1] = q.y; u.w[4 * i + 2] = q.z; u.w[4 * i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kWords; ++i) u.w[i] = 0u;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      if (col + i < cols) {
        if constexpr (DT == kF32) u.w[i] = static_cast<const uint32_t*>(row)[col + i];
        else u.w[i >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(row)[col + i]) << (16 * (i & 1));
      }
    }
  }
  return u;
}

// The bits of the largest magnitude, as fp32 (a NaN's are above an infinity's).
template <int DT>
__device__ __forceinline__ uint32_t unit_top(const Unit<DT>& u) {
  if constexpr (DT == kF32) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, u.w[i] & 0x7FFFFFFFu);
    return m;
  } else {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, u.w[i] & 0x7FFF7FFFu);
    m = max(m & 0xFFFFu, m >> 16);
    if constexpr (DT == kBF16) return m << 16;
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
  }
}

// Weight scales as they are stored: one a row, or one for all rows (step 0).
struct RowScales {
  const void* scale;
  int32_t dtype;
  int32_t step;
  int32_t over_127;  // values are codes times a row's largest magnitude over 127
};

__device__ __forceinline__ float row_scale(const RowScales& s, int64_t row) {
  const int64_t at = row * s.step;
  const float v = s.dtype == kF32    ? static_cast<const float*>(s.scale)[at]
                  : s.dtype == kBF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(s.scale)[at])
                                     : __half2float(static_cast<const __half*>(s.scale)[at]);
  return s.over_127 != 0 ? __fdiv_rn(v, 127.0f) : v;
}

// The expert that a row belongs to, found by a warp: the first one whose end is past it, ends as they count to find_tile
// (one below an end before it as that end, one past the tokens as theirs); `experts` if there is none.
__device__ __forceinline__ int expert_of(const int32_t* ends, int experts, int row) {
  if (ends == nullptr) return 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int e = e0 + static_cast<int>(threadIdx.x & 31);
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, e < experts && ends[e] > row);
    if (hit != 0u) return e0 + __ffs(hit) - 1;
  }
  return experts;
}

// ------------------------------------------------------------------ rows of threads
// A row is worked on by kWarps warps: one, eight rows a block, or all of a block. A lane holds the first kHold units of its
// row in registers between the maximum and the codes, and reads the others again.
template <int kWarps>
struct RowTeam {
  int64_t row;
  int thread;  // of the row's 32 * kWarps

  __device__ __forceinline__ RowTeam(int64_t block) {
    if constexpr (kWarps == 1) {
      row = block * 8 + (threadIdx.x >> 5);
      thread = threadIdx.x & 31;
    } else {
      row = block;
      thread = threadIdx.x;
    }
  }
  // Of all the row's threads; `words` is shared memory, kWarps words for each function.
  __device__ __forceinline__ uint32_t max_of(uint32_t v, uint32_t* words) const {
    v = __reduce_max_sync(0xFFFFFFFFu, v);
    if constexpr (kWarps == 1) return v;
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_max_sync(0xFFFFFFFFu, words[threadIdx.x & (kWarps - 1)]);
  }
  __device__ __forceinline__ int sum_of(int v, uint32_t* words) const {
    v = __reduce_add_sync(0xFFFFFFFFu, v);
    if constexpr (kWarps == 1) return v;
    if ((threadIdx.x & 31) == 0) words[kWarps + (threadIdx.x >> 5)] = static_cast<uint32_t>(v);
    __syncthreads();
    return __reduce_add_sync(0xFFFFFFFFu, (threadIdx.x & 31) < kWarps ? static_cast<int>(words[kWarps + (threadIdx.x & (kWarps - 1))]) : 0);
  }
};

// ------------------------------------------------------------------------- tokens
struct QuantArgs {
  const void* x;
  int64_t x_stride;
  int64_t tokens;
  int32_t cols;
  int64_t pitch;   // bytes between rows of codes, a multiple of 16
  int8_t* codes;
  float* scale;    // (tokens)
  int32_t* sums;   // (tokens) sums of codes, or NULL
};

// What turns a row's values into codes.
struct Quotient {
  float up;       // 127 times a power of two that takes the row's maximum `top` from the ends of fp32's range
  float top;      // the maximum times that power
  float inverse;  // 1 / top, or 0
  float scale;    // of the codes
};

__device__ __forceinline__ Quotient quotient_of(uint32_t top_bits) {
  const float a = __uint_as_float(top_bits);
  const float power = a >= 0x1p64f ? 0x1p-64f : a < 0x1p-64f ? 0x1p64f : 1.0f;
  Quotient q;
  q.up = 127.0f * power;
  q.top = a * power;
  q.inverse = a > 0.0f ? __fdiv_rn(1.0f, q.top) : 0.0f;
  q.scale = a < INFINITY ? __fdiv_rn(a, 127.0f) : NAN;
  return q;
}

constexpr float kRint = 12582912.0f;  // 1.5 * 2^23: added to a small number it leaves its nearest whole one in the low bits

// The bits of kRint plus the code: the code is the low byte.
template <int DT>
__device__ __forceinline__ uint32_t code_bits(float x, const Quotient& q) {
  const float p = x * q.up;
  const float t = p * q.inverse;
  float rest = fmaf(-t, q.top, p);
  if constexpr (DT == kF32) rest += fmaf(x, q.up, -p);  // what the product left
  const float v = fmaf(rest, q.inverse, t);
  const float m = v + kRint;
  if constexpr (DT == kF32) {
    const float whole = m - kRint;
    const float off = v - whole;
    if (fabsf(off) == 0.5f) {
      // the quotient rounds onto a half: 127 x - v top tells on which side it is
      const float left = fmaf(-v, q.top, p) + fmaf(x, q.up, -p);
      const float next = whole + 2.0f * off;  // the other neighbour
      if (left != 0.0f) return __float_as_uint((left > 0.0f ? fmaxf(whole, next) : fminf(whole, next)) + kRint);
    }
  }
  return __float_as_uint(m);
}

template <int DT>
__device__ __forceinline__ int store_codes(const Unit<DT>& u, const Quotient& q, int8_t* to) {
  uint32_t w[4];
  int sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = code_bits<DT>(unit_value<DT>(u, 4 * i + k), q);
    w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    sum = __dp4a(static_cast<int>(w[i]), 0x01010101, sum);
  }
  *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
  return sum;
}

// One or eight rows. Codes behind the last column are zero up to the pitch.
template <int DT, int kWarps, int kHold, bool kVec>
__device__ __forceinline__ void quantize_rows(const QuantArgs& p, int64_t block, uint32_t* words) {
  const RowTeam<kWarps> team(block);
  if (kWarps == 1 && team.row >= p.tokens) return;
  constexpr int kStep = 32 * kWarps;
  const uint8_t* row = static_cast<const uint8_t*>(p.x) + team.row * p.x_stride * (DT == kF32 ? 4 : 2);
  const int units = static_cast<int>(p.pitch / kUnit);
  Unit<DT> held[kHold];
  uint32_t top = 0u;
#pragma unroll
  for (int k = 0; k < kHold; ++k)
    if (team.thread + k * kStep < units) held[k] = load_unit<DT, kVec>(row, (team.thread + k * kStep) * kUnit, p.cols);
#pragma unroll
  for (int k = 0; k < kHold; ++k)
    if (team.thread + k * kStep < units) top = max(top, unit_top<DT>(held[k]));
  for (int u = team.thread + kHold * kStep; u < units; u += kStep) top = max(top, unit_top<DT>(load_unit<DT, kVec>(row, u * kUnit, p.cols)));
  const Quotient q = quotient_of(team.max_of(top, words));
  int8_t* to = p.codes + team.row * p.pitch;
  int sum = 0;
#pragma unroll
  for (int k = 0; k < kHold; ++k)
    if (team.thread + k * kStep < units) sum += store_codes<DT>(held[k], q, to + (team.thread + k * kStep) * kUnit);
  for (int u = team.thread + kHold * kStep; u < units; u += kStep)
    sum += store_codes<DT>(load_unit<DT, kVec>(row, u * kUnit, p.cols), q, to + u * kUnit);
  if (p.sums != nullptr) sum = team.sum_of(sum, words);
  if (team.thread == 0) {
    p.scale[team.row] = q.scale;
    if (p.sums != nullptr) p.sums[team.row] = sum;
  }
}

// ---------------------------------------------------------------------- gradients
// dy[t, n] times the scale of the weight's row n, times a power of two of row t that brings its largest value to
// [2^14, 2^15), as fp16: 11 bits, an eighth of bf16's rounding and as many as an fp16 gradient has itself, and exact for the
// rest of the product, whose other factor has 9 bits. What is more than 2^29 below the row's largest value is rounded at
// 2^-40 of it. fp32 gradients are two such terms, each the rounding of what the one before it left: 22 bits and a sign. Two
// for all types would take twice the products (1024 x 4096 x 4096 65 us, 36 with one). With one the result of 512 x 4096 x 1024
// is off by 1.67e-3 of its norm for bf16, of which its own rounding is 1.66e-3, and by 2.9e-4 for fp16, rounding 2.1e-4.
struct ScaleArgs {
  const void* dy;
  int64_t dy_stride;
  int64_t tokens;
  int32_t rows;    // of one weight: values in a row of dy
  int64_t pitch;   // values between rows of out, a multiple of 16
  __half* out;     // (terms, tokens, pitch)
  float* back;     // (tokens): what a row's sums are multiplied by
  RowScales scales;
  const int32_t* ends;
  int32_t experts;
};

// Sixteen values times the scales of the weight's rows from `n` on, 0 past the last. A lane takes scales as it takes values.
template <int DT, int SDT, bool kVec>
__device__ __forceinline__ void scaled_unit(const ScaleArgs& p, const Unit<DT>& u, int64_t row0, int n, float (&v)[kUnit]) {
  if (p.scales.step == 0) {
    const float one = row_scale(p.scales, 0);
#pragma unroll
    for (int i = 0; i < kUnit; ++i) v[i] = n + i < p.rows ? unit_value<DT>(u, i) * one : 0.0f;
    return;
  }
  const Unit<SDT> s = load_unit<SDT, kVec>(static_cast<const uint8_t*>(p.scales.scale) + row0 * (SDT == kF32 ? 4 : 2), n, p.rows);
#pragma unroll
  for (int i = 0; i < kUnit; ++i) {
    const float scale = unit_value<SDT>(s, i);
    v[i] = unit_value<DT>(u, i) * (p.scales.over_127 != 0 ? __fdiv_rn(scale, 127.0f) : scale);
  }
}

// A row whose values lie at `row`, the first units in `held`. Products are made once for their maximum and once to be
// written, with scales from L1: kept in between they would take twice the registers of the values.
template <int DT, int SDT, int kWarps, int kHold, bool kVec>
__device__ __forceinline__ void scale_row(const ScaleArgs& p, const RowTeam<kWarps>& team, const uint8_t* row, const Unit<DT> (&held)[kHold],
                                          int64_t row0, int units, uint32_t* words) {
  constexpr int kStep = 32 * kWarps;
  // of unit k of this lane, one of the row's last units again where it has no more
  const auto products = [&](int k, float (&v)[kUnit]) {
    const int n = min(team.thread + k * kStep, units - 1) * kUnit;
    if (k < kHold) scaled_unit<DT, SDT, kVec>(p, held[k], row0, n, v);
    else scaled_unit<DT, SDT, kVec>(p, load_unit<DT, kVec>(row, n, p.rows), row0, n, v);
  };
  // the largest magnitude that is a number; infinities only cost a second look
  const auto largest = [&](bool finite) {
    float top = 0.0f;
    const auto see = [&](const float (&v)[kUnit]) {
#pragma unroll
      for (int i = 0; i < kUnit; ++i) top = fmaxf(top, finite && !(fabsf(v[i]) < INFINITY) ? 0.0f : fabsf(v[i]));  // a NaN is not counted
    };
    float v[kUnit];
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      products(k, v);
      see(v);
    }
    for (int k = kHold; team.thread + k * kStep < units; ++k) {
      products(k, v);
      see(v);
    }
    return team.max_of(__float_as_uint(top), words);
  };
  uint32_t bits = largest(false);
  if (bits == __float_as_uint(INFINITY)) {
    if constexpr (kWarps > 1) __syncthreads();  // the words are read
    bits = largest(true);
  }
  // 2^(14 - exponent), within fp32's normal numbers; 1 for a row of zeros
  const int exponent = bits == 0u ? 14 : max(static_cast<int>(bits >> 23) - 127, -112);
  const float power = __uint_as_float(static_cast<uint32_t>(141 - exponent) << 23);
  const auto write = [&](int k) {
    float v[kUnit];
    products(k, v);
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < kUnit; i += 2) {
      const float a = v[i] * power, b = v[i + 1] * power;
      const __half2 h = __floats2half2_rn(a, b);
      hi[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
      if constexpr (DT == kF32) {
        // an infinity or a NaN is its first term alone
        const __half2 l = __floats2half2_rn(fabsf(a) < INFINITY ? a - __low2float(h) : 0.0f, fabsf(b) < INFINITY ? b - __high2float(h) : 0.0f);
        lo[i / 2] = *reinterpret_cast<const uint32_t*>(&l);
      }
    }
    const int64_t at = static_cast<int64_t>(team.thread + k * kStep) * kUnit;
    uint4* to = reinterpret_cast<uint4*>(p.out + team.row * p.pitch + at);
    to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    to[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
    if constexpr (DT == kF32) {
      to = reinterpret_cast<uint4*>(p.out + (p.tokens + team.row) * p.pitch + at);
      to[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      to[1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
    }
  };
#pragma unroll
  for (int k = 0; k < kHold; ++k)
    if (team.thread + k * kStep < units) write(k);
  for (int k = kHold; team.thread + k * kStep < units; ++k) write(k);
  if (team.thread == 0) p.back[team.row] = __uint_as_float(static_cast<uint32_t>(113 + exponent) << 23);
}

template <int DT, int kWarps, int kHold, bool kVec>
__device__ __forceinline__ void scale_rows(const ScaleArgs& p, int64_t block, uint32_t* words) {
  const RowTeam<kWarps> team(block);
  if (kWarps == 1 && team.row >= p.tokens) return;
  const uint8_t* row = static_cast<const uint8_t*>(p.dy) + team.row * p.dy_stride * (DT == kF32 ? 4 : 2);
  const int units = static_cast<int>(p.pitch / kUnit);
  Unit<DT> held[kHold];  // under way while the expert is found
#pragma unroll
  for (int k = 0; k < kHold; ++k) held[k] = load_unit<DT, kVec>(row, min(team.thread + k * 32 * kWarps, units - 1) * kUnit, p.rows);
  const int expert = expert_of(p.ends, p.experts, static_cast<int>(team.row));
  if (expert == p.experts) return;  // a row of no expert
  const int64_t row0 = static_cast<int64_t>(expert) * p.rows;
  if (p.scales.dtype == kBF16) scale_row<DT, kBF16, kWarps, kHold, kVec>(p, team, row, held, row0, units, words);
  else if (p.scales.dtype == kF16) scale_row<DT, kF16, kWarps, kHold, kVec>(p, team, row, held, row0, units, words);
  else scale_row<DT, kF32, kWarps, kHold, kVec>(p, team, row, held, row0, units, words);
}

// -------------------------------------------------------------------------- codes
// Codes whose rows do not start on 16-byte boundaries, which bulk copies need, laid out so. A thread makes 16 bytes.
struct RepackArgs {
  const uint8_t* codes;
  uint8_t* out;
  int64_t cols;    // bytes of a row
  int64_t pitch;   // of out, a multiple of 16
  int64_t pieces;  // 16-byte pieces of out
};

__device__ __forceinline__ void repack(const RepackArgs& p, int64_t piece) {
  if (piece >= p.pieces) return;
  const int64_t per = p.pitch / 16, row = piece / per, col = (piece - row * per) * 16;
  // aligned words that hold the bytes, shifted into place; none is read that holds no byte of the row
  const uintptr_t from = reinterpret_cast<uintptr_t>(p.codes) + static_cast<uintptr_t>(row * p.cols + col);
  const int64_t bytes = min(static_cast<int64_t>(16), p.cols - col);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(from & ~uintptr_t{3});
  const uint32_t shift = static_cast<uint32_t>(from & 3);
  uint32_t in[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) in[i] = i * 4 < bytes + shift ? words[i] : 0u;
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i] = __funnelshift_r(in[i], in[i + 1], shift * 8);
    const int64_t left = bytes - i * 4;
    if (left < 4) out[i] &= left <= 0 ? 0u : (1u << (8 * left)) - 1u;
  }
  *reinterpret_cast<uint4*>(p.out + piece * 16) = make_uint4(out[0], out[1], out[2], out[3]);
}

// The launch before a product: blocks of token rows, then of codes.
template <int DT, int kWarps, int kHold, bool kVec>
__global__ void __launch_bounds__(prepare_threads(kWarps)) quantize_kernel(const __grid_constant__ QuantArgs q, const __grid_constant__ RepackArgs r,
                                                                   uint32_t token_blocks) {
  __shared__ uint32_t words[2 * kWarps];
  // in this order: the product that follows reads the ends of groups and loads its weight as soon as it begins
  fp4::grid_wait();
  fp4::grid_launch_dependents();
  if (blockIdx.x < token_blocks) quantize_rows<DT, kWarps, kHold, kVec>(q, blockIdx.x, words);
  else repack(r, static_cast<int64_t>(blockIdx.x - token_blocks) * prepare_threads(kWarps) + threadIdx.x);
}

// The launch before a gradient.
template <int DT, int kWarps, int kHold, bool kVec>
__global__ void __launch_bounds__(prepare_threads(kWarps)) scale_kernel(const __grid_constant__ ScaleArgs s, const __grid_constant__ RepackArgs r,
                                                                uint32_t token_blocks) {
  __shared__ uint32_t words[2 * kWarps];
  fp4::grid_wait();  // first, as in quantize_kernel
  fp4::grid_launch_dependents();
  if (blockIdx.x < token_blocks) scale_rows<DT, kWarps, kHold, kVec>(s, blockIdx.x, words);
  else repack(r, static_cast<int64_t>(blockIdx.x - token_blocks) * prepare_threads(kWarps) + threadIdx.x);
}

}  // namespace i8
