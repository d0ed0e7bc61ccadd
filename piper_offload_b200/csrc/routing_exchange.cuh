// routing_exchange.cuh - tokens to their places among the experts' rows, and the experts' rows added up again.
//
// All of it is memory: every row is read once and written once, 16 bytes a thread where rows start on 16-byte boundaries
// (one value otherwise). A place past the last end counts as none. 8,192 tokens of 2,048 bf16 to eight experts each: copies
// 48 us (6.2 TB/s of what it reads and writes), sums 51 us (5.9), both gradients of the sums 105 (5.4).
#pragma once
#include "routing_route.cuh"

namespace routing {

constexpr int kExchangeThreads = 256;

struct ExchangeArgs {
  const void* in;        // dispatch: tokens; combine: rows
  int64_t in_stride;
  const void* dout;      // combine's gradient: of its result
  int64_t dout_stride;
  const float* weights;  // or NULL: ones
  void* out;
  float* dweights;
  const int32_t* rows;   // (tokens, top_k)
  const int32_t* total;
  int64_t tokens;
  int32_t top_k, hidden;
  int32_t pieces;        // of a row
};

// V values of a row at once, as they lie.
template <int DT, int V>
struct Pack {
  static constexpr int kWords = V * (DT == kF32 ? 4 : 2) / 4;
  uint32_t w[kWords > 0 ? kWords : 1];
};

template <int DT, int V>
__device__ __forceinline__ Pack<DT, V> load_pack(const void* p, int64_t at) {
  Pack<DT, V> r;
  if constexpr (V == 1) {
    if constexpr (DT == kF32) r.w[0] = static_cast<const uint32_t*>(p)[at];
    else r.w[0] = static_cast<const uint16_t*>(p)[at];
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (DT == kF32 ? 4 : 2));
    r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
  }
  return r;
}

// The same, of what nothing reads again: it leaves the cache first.
template <int DT, int V>
__device__ __forceinline__ Pack<DT, V> load_pack_once(const void* p, int64_t at) {
  if constexpr (V == 1) return load_pack<DT, V>(p, at);
  Pack<DT, V> r;
  const uint4 q = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (DT == kF32 ? 4 : 2)));
  r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
  return r;
}

template <int DT, int V>
__device__ __forceinline__ void store_pack(void* p, int64_t at, const Pack<DT, V>& r) {
  if constexpr (V == 1) {
    if constexpr (DT == kF32) static_cast<uint32_t*>(p)[at] = r.w[0];
    else static_cast<uint16_t*>(p)[at] = static_cast<uint16_t>(r.w[0]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p) + at * (DT == kF32 ? 4 : 2)) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  }
}

template <int DT, int V>
__device__ __forceinline__ void to_floats(const Pack<DT, V>& r, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (DT == kF32) f[i] = __uint_as_float(r.w[i]);
    else {
      const uint32_t h = r.w[i >> 1] >> (16 * (i & 1)) & 0xFFFFu;
      if constexpr (DT == kBF16) f[i] = __uint_as_float(h << 16);
      else f[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
    }
  }
}

template <int DT, int V>
__device__ __forceinline__ Pack<DT, V> from_floats(const float (&f)[V]) {
  Pack<DT, V> r{};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (DT == kF32) r.w[i] = __float_as_uint(f[i]);
    else {
      const uint32_t h = DT == kBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f[i])) : __half_as_ushort(__float2half_rn(f[i]));
      r.w[i >> 1] |= h << (16 * (i & 1));
    }
  }
  return r;
}

// The place of choice j of a token, or -1. `places`: of all choices, of which there are fewer than 2^31.
__device__ __forceinline__ int32_t place_of(const ExchangeArgs& p, int32_t places, int64_t token, int j) {
  const int32_t r = p.rows[token * p.top_k + j];
  return r >= 0 && r < places ? r : -1;
}

// The places that have a choice, as the ends of experts tell.
__device__ __forceinline__ int32_t places_of(const ExchangeArgs& p) {
  return static_cast<int32_t>(min(static_cast<int64_t>(*p.total), p.tokens * p.top_k));
}

// A thread has a piece of a token. It writes the copies, and zeros in the rows of no choice among [t top_k, (t + 1) top_k).
template <int DT, int V>
__global__ void __launch_bounds__(kExchangeThreads) dispatch_kernel(const __grid_constant__ ExchangeArgs p) {
  fp4::grid_launch_dependents();
  fp4::grid_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kExchangeThreads + threadIdx.x;
  const int64_t token = i / p.pieces;
  if (token >= p.tokens) return;
  const int64_t col = (i - token * p.pieces) * V;
  const Pack<DT, V> v = load_pack<DT, V>(p.in, token * p.in_stride + col);
  const int32_t total = places_of(p);
  for (int j = 0; j < p.top_k; ++j) {
    const int32_t r = place_of(p, total, token, j);
    if (r >= 0) store_pack<DT, V>(p.out, static_cast<int64_t>(r) * p.hidden + col, v);
    if (token * p.top_k + j >= total) store_pack<DT, V>(p.out, (token * p.top_k + j) * p.hidden + col, Pack<DT, V>{});
  }
}

constexpr int kAtOnce = 8;  // loads of rows that a thread has in flight: of K choices for each of kAtOnce / K pieces

// A thread has kAtOnce / K pieces of tokens' results. Of eight choices the rows leave the cache first (8,192 tokens of 8 x
// 2,048 bf16: 51 us, 56 without; 8,192 of 6 x 1,000: 24 and 27), of fewer not (4,096 of 4 x 4,096: 37 with, 36 without).
template <int DT, int V, int K>
__global__ void __launch_bounds__(kExchangeThreads, K == 8 ? 4 : K == 4 ? 3 : 2) combine_kernel(const __grid_constant__ ExchangeArgs p) {
  fp4::grid_launch_dependents();
  fp4::grid_wait();
  constexpr int kPieces = kAtOnce / K;
  int64_t token[kPieces], col[kPieces];
  float sum[kPieces][V];
#pragma unroll
  for (int q = 0; q < kPieces; ++q) {
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * kPieces + q) * kExchangeThreads + threadIdx.x;
    token[q] = i / p.pieces;
    col[q] = (i - token[q] * p.pieces) * V;
#pragma unroll
    for (int k = 0; k < V; ++k) sum[q][k] = 0.0f;
  }
  const int32_t total = places_of(p);
  for (int j0 = 0; j0 < p.top_k; j0 += K) {
    Pack<DT, V> v[kPieces][K];
    float w[kPieces][K];
    bool has[kPieces][K];
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int32_t r = token[q] < p.tokens && j0 + k < p.top_k ? place_of(p, total, token[q], j0 + k) : -1;
        has[q][k] = r >= 0;
        if (r >= 0) {
          const int64_t at = static_cast<int64_t>(r) * p.in_stride + col[q];
          v[q][k] = K == 8 ? load_pack_once<DT, V>(p.in, at) : load_pack<DT, V>(p.in, at);
          w[q][k] = p.weights != nullptr ? p.weights[token[q] * p.top_k + j0 + k] : 1.0f;
        }
      }
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (has[q][k]) {
          float f[V];
          to_floats(v[q][k], f);
#pragma unroll
          for (int n = 0; n < V; ++n) sum[q][n] = fmaf(w[q][k], f[n], sum[q][n]);
        }
  }
#pragma unroll
  for (int q = 0; q < kPieces; ++q)
    if (token[q] < p.tokens) store_pack<DT, V>(p.out, token[q] * p.hidden + col[q], from_floats<DT, V>(sum[q]));
}

// kWarps warps have a token: each piece of the result's gradient goes to the rows' gradients, and with the rows into the
// weights' gradients. Blocks an SM: with eight choices more than two cost registers that the loads in flight need (8,192
// tokens of 8 x 2,048 bf16: 105 us with two, 113 with three); fewer choices gain (4,096 of 4 x 4,096: 48 with four, 51 with
// three, 59 with two), and so do single values (3,000 of 8 x 2,047: 80 with three, 93 with four, 114 with two).
template <int DT, int V, int K, int kWarps>
__global__ void __launch_bounds__(kExchangeThreads, V == 1 ? 3 : K == 8 ? 2 : 4) combine_grad_kernel(const __grid_constant__ ExchangeArgs p) {
  fp4::grid_launch_dependents();
  fp4::grid_wait();
  constexpr int kPieces = kAtOnce / K, kStep = 32 * kWarps;
  __shared__ float parts[kWarps > 1 ? K * 8 : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t token = kWarps == 1 ? static_cast<int64_t>(blockIdx.x) * (kExchangeThreads / 32) + warp : blockIdx.x;
  if (kWarps == 1 && token >= p.tokens) return;
  const int first = kWarps == 1 ? lane : threadIdx.x;
  const int32_t total = places_of(p);
  for (int j0 = 0; j0 < p.top_k; j0 += K) {
    int32_t row[K];
    float w[K], dot[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool in = j0 + k < p.top_k;
      row[k] = in ? place_of(p, total, token, j0 + k) : -1;
      w[k] = in ? p.weights[token * p.top_k + j0 + k] : 0.0f;
      dot[k] = 0.0f;
    }
    for (int piece0 = first; piece0 < p.pieces; piece0 += kStep * kPieces) {
      Pack<DT, V> d[kPieces], y[kPieces][K];
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        const int piece = piece0 + q * kStep;
        if (piece >= p.pieces) continue;
        d[q] = load_pack<DT, V>(p.dout, token * p.dout_stride + static_cast<int64_t>(piece) * V);
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (row[k] >= 0) y[q][k] = load_pack<DT, V>(p.in, static_cast<int64_t>(row[k]) * p.in_stride + static_cast<int64_t>(piece) * V);
      }
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        const int piece = piece0 + q * kStep;
        if (piece >= p.pieces) continue;
        const int64_t col = static_cast<int64_t>(piece) * V;
        float g[V];
        to_floats(d[q], g);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (row[k] >= 0) {
            float f[V], dy[V];
            to_floats(y[q][k], f);
#pragma unroll
            for (int n = 0; n < V; ++n) {
              dot[k] = fmaf(f[n], g[n], dot[k]);
              dy[n] = w[k] * g[n];
            }
            store_pack<DT, V>(p.out, static_cast<int64_t>(row[k]) * p.hidden + col, from_floats<DT, V>(dy));
          }
          const int64_t none = token * p.top_k + j0 + k;
          if (j0 + k < p.top_k && none >= total) store_pack<DT, V>(p.out, none * p.hidden + col, Pack<DT, V>{});
        }
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) dot[k] = warp_sum(dot[k]);
    if constexpr (kWarps > 1) {
      __syncthreads();  // the last ones are read
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (lane == 0) parts[k * 8 + warp] = dot[k];
      __syncthreads();
      if (threadIdx.x < K && j0 + static_cast<int>(threadIdx.x) < p.top_k) {
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < kWarps; ++n) sum += parts[threadIdx.x * 8 + n];
        p.dweights[token * p.top_k + j0 + threadIdx.x] = sum;
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (lane == k && j0 + k < p.top_k) p.dweights[token * p.top_k + j0 + k] = dot[k];
    }
  }
}

}  // namespace routing
