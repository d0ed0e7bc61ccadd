// routing_route.cuh - a token's experts: scores, the best groups, the best experts in them, weights, and the order by expert.
//
// A warp has a token and each lane N neighbouring experts. Choices are compared as whole numbers that order as the scores
// do (0 for what is closed, 1 for a NaN): the largest is found by redux, its lane by a vote, so that ties go to the lowest
// index.
//
// With up to eight experts a lane (choose_quickly) a key's last three bits give way to the expert's place in the lane, so
// that a lane sorts its keys by 19 minima and maxima and keeps the list in shared memory; a round then is a redux, a vote
// and one load by the lane whose largest is taken. Groups whose experts fill a power of two of lanes are compared all at
// once by shuffles. What this leaves open is decided in 64 bits: between groups over all their experts, between the
// experts next to each other over those alone, a lane each. Only what that cannot separate (more than 32 scores next to
// each other) is done again as a whole, in choose(). Open are
// - Choice scores. Without a bias the logits decide, since both scores grow with them. With one, or where a group counts by
//   its two best, sums of scores do, and sums near each other in fp32 may be in another order than the numbers they stand
//   for. Each gap that decides anything is held against 2^-16, which is above twice the error of two scores added up: they
//   are at most 1 (of sigmoids 2), the fast exponential is off by 2 steps of 2^-23 and 1.2 more for each unit of its
//   argument d, where d exp(-d) is below 0.37, the fast quotient by 2 steps, a softmax's sum by a step of 2^-24 for each of
//   at most 37 additions, the cut of three bits by 8 steps of 2^-24 for the sum; together below 2^-17.5. Where scores of
//   logits are added up they are made of the whole logits: a softmax's error by three bits of a logit grows with the logit,
//   whatever the score (7 steps of 2^-14 at 1000; 1.4 us of 34.6 without a bias for 16,384 x 256). 2^-19 of the
//   sum is above twice its rounding and cut. A group's two best may cancel (biases of +1000 and -1000), so its bounds are
//   half of 2^-16 and 9 steps of 2^-23 of what was added up: 7 of them cut, a half each for the sum with the bias, for that
//   of the two and for the bound's own. 256 experts' scores spread over [0, 1]
//   leave 1 % of the tokens open; all of such a token done again by one warp in 64 bits took 8 us, while its block waited.
// - fp32 logits that are equal but for the last three bits (16-bit ones lose nothing).
//
// The order by expert is two steps: a block counts its tokens' choices by expert, and when all have, every block adds up the
// counts of the chunks before its own and places its choices. Up to 128 tokens are one launch of one block (64 x 8 logits
// 7.4 us), else two: 16,384 x 256 fp32 logits in eight groups take 36 us, of which reading them is 3 and issue most of the
// rest; 777 x 60 take 8, launches and latency. The gradient reads what was chosen again: 9 and 4 us.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "fp4_ptx.cuh"

namespace routing {

enum : int { kBF16 = 0, kF16 = 1, kF32 = 2 };
enum : int { kSoftmax = 0, kSigmoid = 1 };
enum : int { kMax = 0, kTop2 = 1 };

constexpr uint32_t kFull = 0xFFFFFFFFu;

struct RouteArgs {
  const void* logits;
  int64_t stride;
  const float* bias;
  const uint8_t* mask;
  float* weights;
  int32_t* experts_out;
  int32_t* ends;
  int32_t* rows;
  int32_t* source;
  int32_t* counts;  // (chunks, pitch)
  int64_t tokens;
  int32_t chunk;    // tokens of a block
  int32_t chunks;
  int32_t experts, top_k;
  int32_t pitch;    // experts up to a multiple of four
  int32_t scoring, groups, top_groups, group_score, renormalize;
  int32_t quick;    // choose_quickly() takes the groups
  int32_t vec, bias_vec;  // a lane's logits, or biases, may be read in pieces of 16 bytes, or of all its bytes
  float scale;
};

template <int DT>
__device__ __forceinline__ float value_at(const void* p, int64_t at) {
  if constexpr (DT == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  else if constexpr (DT == kF16) return __half2float(static_cast<const __half*>(p)[at]);
  else return static_cast<const float*>(p)[at];
}

// A lane's N neighbouring values of a row, from value `at` on; -infinity past the last.
template <int DT, int N>
__device__ __forceinline__ void load_values(const void* from, int64_t at, int count, bool vec, float (&v)[N]) {
  constexpr int kSize = DT == kF32 ? 4 : 2, kBytes = N * kSize < 16 ? N * kSize : 16, kEach = kBytes / kSize;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = -INFINITY;
  if (vec && kBytes >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += kEach) {
      if (i >= count) continue;  // a piece is there or not as a whole
      uint32_t w[kBytes >= 4 ? kBytes / 4 : 1];
      const uint8_t* q = static_cast<const uint8_t*>(from) + (at + i) * kSize;
      if constexpr (kBytes == 16) {
        const uint4 r = *reinterpret_cast<const uint4*>(q);
        w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
      } else if constexpr (kBytes == 8) {
        const uint2 r = *reinterpret_cast<const uint2*>(q);
        w[0] = r.x; w[1] = r.y;
      } else {
        w[0] = *reinterpret_cast<const uint32_t*>(q);
      }
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        if constexpr (DT == kF32) v[i + k] = __uint_as_float(w[k]);
        else if constexpr (DT == kBF16) v[i + k] = __uint_as_float(k & 1 ? w[k >> 1] & 0xFFFF0000u : w[k >> 1] << 16);
        else v[i + k] = __half2float(__ushort_as_half(static_cast<unsigned short>(w[k >> 1] >> (16 * (k & 1)))));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < count) v[i] = value_at<DT>(from, at + i);
  }
}

// ------------------------------------------------------------------ numbers that order as values do
template <class T>
struct Order;
template <>
struct Order<float> {
  using Key = uint32_t;
  static __device__ __forceinline__ Key of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
    const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return v == v ? k : 1u;
  }
  static __device__ __forceinline__ float value(Key k) {
    return k == 1u ? NAN : __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
  }
  static __device__ __forceinline__ Key max_of(Key k) { return __reduce_max_sync(kFull, k); }
  static __device__ __forceinline__ Key from(Key k, int lane) { return __shfl_sync(kFull, k, lane); }
};
template <>
struct Order<double> {
  using Key = uint64_t;
  static __device__ __forceinline__ Key of(double v) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    const uint64_t k = b ^ (static_cast<uint64_t>(static_cast<int64_t>(b) >> 63) | 0x8000000000000000ull);
    return v == v ? k : 1u;
  }
  static __device__ __forceinline__ double value(Key k) {
    return k == 1u ? static_cast<double>(NAN) : __longlong_as_double(static_cast<int64_t>(k >> 63 ? k ^ 0x8000000000000000ull : ~k));
  }
  static __device__ __forceinline__ Key max_of(Key k) {
    const uint32_t hi = static_cast<uint32_t>(k >> 32), top = __reduce_max_sync(kFull, hi);
    return static_cast<Key>(top) << 32 | __reduce_max_sync(kFull, hi == top ? static_cast<uint32_t>(k) : 0u);
  }
  static __device__ __forceinline__ Key from(Key k, int lane) { return __shfl_sync(kFull, k, lane); }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// For scores that are compared: the fast forms in fp32 (the margin below covers them).
__device__ __forceinline__ float exp_of(float v) { return __expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float quotient(float a, float b) { return __fdividef(a, b); }
__device__ __forceinline__ double quotient(double a, double b) { return a / b; }

// What a token's row of logits has: the largest (a NaN not counted), and whether one is a NaN or +infinity, for which
// softmax is a NaN everywhere.
struct Row {
  float top;
  bool broken;
};

// Whether sums of scores decide anything, or the logits alone.
__device__ __forceinline__ bool scores_decide(const RouteArgs& p) { return p.bias != nullptr || (p.groups > 1 && p.group_score == kTop2); }

constexpr float kMargin = 0x1p-16f, kMarginOfValue = 0x1p-19f, kErrorOfParts = 9 * 0x1p-23f;

// Whether a value is so near one below it that fp32 may have put them in the wrong order. False for what is closed.
__device__ __forceinline__ bool near_by(uint32_t upper, uint32_t lower) {
  if (upper == 0u || lower == 0u) return false;
  const float a = Order<float>::value(upper), b = Order<float>::value(lower);
  return !(a - b > kMargin + kMarginOfValue * fmaxf(fabsf(a), fabsf(b)));
}

// Whether the numbers of a kept group and of one that is not may be in another order than their fp32 keys. A lane has a group's
// key (0 for none, and for one with nothing open) and the magnitudes that it was added up of.
__device__ __forceinline__ bool groups_near(uint32_t own, bool kept, float size) {
  const float v = Order<float>::value(own), off = 0.5f * kMargin + kErrorOfParts * size;
  const uint32_t lowest = __reduce_min_sync(kFull, !kept ? 0xFFFFFFFFu : own == 0u ? 0u : Order<float>::of(v - off));
  const uint32_t highest = __reduce_max_sync(kFull, kept || own == 0u ? 0u : Order<float>::of(v + off));
  return lowest != 0u && highest != 0u && !(Order<float>::value(lowest) > Order<float>::value(highest));
}

// The two largest of a group's keys, as it counts: the best one, or both added up; 0 for a group with nothing open.
template <class T>
__device__ __forceinline__ typename Order<T>::Key group_key(int group_score, typename Order<T>::Key best, typename Order<T>::Key second) {
  using O = Order<T>;
  return group_score == kMax || second == 0 ? best : O::of(O::value(best) + O::value(second));
}

template <class K>
__device__ __forceinline__ void take(K& best, K& second, K k) {
  const K low = k < best ? k : best;
  second = low > second ? low : second;
  best = k > best ? k : best;
}

// Lane j's expert of the token's choice j, or -1; for any number of experts and groups. `near`: in fp32, whether some order is
// not certain.
template <class T, int N>
__device__ __forceinline__ int choose(const RouteArgs& p, const float (&logit)[N], const Row& row, int lane, bool& near) {
  using O = Order<T>;
  using Key = typename O::Key;
  constexpr bool kCheck = sizeof(T) == 4;
  near = false;
  const bool by_score = scores_decide(p);
  const int e0 = lane * N;
  Key choice[N], part[N];  // part: what a group counts by
  if (by_score) {
    T score[N];
    if (p.scoring == kSigmoid) {
#pragma unroll
      for (int i = 0; i < N; ++i) score[i] = quotient(static_cast<T>(1), static_cast<T>(1) + exp_of(-static_cast<T>(logit[i])));
    } else {
      T sum = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        score[i] = exp_of(static_cast<T>(logit[i]) - static_cast<T>(row.top));  // 0 where there is no expert
        sum += score[i];
      }
      sum = warp_sum(sum);
#pragma unroll
      for (int i = 0; i < N; ++i) score[i] = row.broken ? static_cast<T>(NAN) : quotient(score[i], sum);
    }
    if (p.bias != nullptr) {
      float bias[N];
      load_values<kF32, N>(p.bias, e0, p.experts - e0, p.bias_vec != 0, bias);
#pragma unroll
      for (int i = 0; i < N; ++i)
        part[i] = choice[i] = logit[i] != -INFINITY && bias[i] != -INFINITY ? O::of(score[i] + static_cast<T>(bias[i])) : 0;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        part[i] = logit[i] != -INFINITY ? O::of(score[i]) : 0;
        choice[i] = logit[i] != -INFINITY ? O::of(static_cast<T>(logit[i])) : 0;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = choice[i] = logit[i] != -INFINITY ? O::of(static_cast<T>(logit[i])) : 0;
  }

  if (p.groups > 1) {
    const int per = p.experts / p.groups;
    Key own = 0;  // of group `lane`
    float size = 0.0f;
    for (int g = 0; g < p.groups; ++g) {
      Key best = 0, second = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e0 + i >= g * per && e0 + i < g * per + per) take(best, second, p.group_score == kTop2 ? part[i] : choice[i]);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const Key b = __shfl_xor_sync(kFull, best, o), s = __shfl_xor_sync(kFull, second, o);
        take(best, second, b);
        take(best, second, s);
      }
      if (lane == g) {
        own = group_key<T>(p.group_score, best, second);
        if constexpr (kCheck) size = fabsf(O::value(best)) + (p.group_score == kMax || second == 0 ? 0.0f : fabsf(O::value(second)));
      }
    }
    int before = 0;  // groups that come before this lane's
    for (int g = 0; g < p.groups; ++g) {
      const Key other = O::from(own, g);
      before += other > own || (other == own && g < lane);
    }
    const bool kept = lane < p.groups && before < p.top_groups;
    if (kCheck && by_score && p.top_groups < p.groups) near |= groups_near(static_cast<uint32_t>(own), kept, size);
    const uint32_t groups_kept = __ballot_sync(kFull, kept);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (e0 + i < p.experts && !(groups_kept >> ((e0 + i) / per) & 1u)) choice[i] = 0;
  }

  int chosen = -1;
  Key mine = 0;  // of this lane's choice
  Key next = 0;  // the largest that was not chosen
  const int rounds = p.top_k + (kCheck && p.bias != nullptr);  // one more to see how near the next one is
  for (int j = 0; j < rounds; ++j) {
    Key best = choice[0];
    int place = e0;
#pragma unroll
    for (int i = 1; i < N; ++i) {
      place = choice[i] > best ? e0 + i : place;
      best = choice[i] > best ? choice[i] : best;
    }
    const Key top = O::max_of(best);
    if (j == p.top_k) next = top;
    if (top == 0 || j == p.top_k) break;
    const int expert = __shfl_sync(kFull, place, __ffs(__ballot_sync(kFull, best == top)) - 1);
    if (lane == j) {
      chosen = expert;
      mine = top;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) choice[i] = e0 + i == expert ? 0 : choice[i];
  }
  if (kCheck && p.bias != nullptr) {
    const Key below = __shfl_down_sync(kFull, mine, 1);
    near |= __any_sync(kFull, near_by(static_cast<uint32_t>(mine), static_cast<uint32_t>(lane + 1 == p.top_k ? next : lane == 31 ? 0 : below)));
  }
  return chosen;
}

template <class T, int N>
__device__ __noinline__ int choose_apart(const RouteArgs& p, const float (&logit)[N], const Row& row, int lane, bool& near) {
  return choose<T, N>(p, logit, row, lane, near);
}

// A warp's sorted lists (choose_quickly): each lane's keys after its largest, and the experts chosen.
template <int N>
struct Lists {
  static constexpr bool kUsed = N <= 8;
  uint32_t key[kUsed ? N : 1][kUsed ? 32 : 1];
  uint16_t chosen[kUsed ? 32 : 2];
};

// The largest key first.
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[N]) {
  constexpr int kPairs = N == 8 ? 19 : N == 4 ? 5 : N == 2 ? 1 : 0;
  constexpr int kFirst[19] = {0, 1, 4, 5, 0, 1, 2, 3, 0, 2, 4, 6, 2, 3, 1, 3, 1, 3, 5}, kSecond[19] = {2, 3, 6, 7, 4, 5, 6, 7, 1, 3, 5, 7, 4, 5, 4, 6, 2, 4, 6};
  constexpr int kFirst4[5] = {0, 2, 0, 1, 1}, kSecond4[5] = {1, 3, 2, 3, 2};
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int a = N == 8 ? kFirst[i] : N == 4 ? kFirst4[i] : 0, b = N == 8 ? kSecond[i] : N == 4 ? kSecond4[i] : 1;
    const uint32_t high = max(k[a], k[b]), low = min(k[a], k[b]);
    k[a] = high;
    k[b] = low;
  }
}

constexpr uint32_t kKeyBits = ~7u;

// A value's key with the expert's place in its lane; 0 for what is closed.
__device__ __forceinline__ uint32_t placed_key(float v, int i, bool open) {
  const uint32_t k = Order<float>::of(v);
  return open ? ((k == 1u ? 8u : k) & kKeyBits) | static_cast<uint32_t>(7 - i) : 0u;
}

__device__ __forceinline__ float key_value(uint32_t k) { return Order<float>::value((k & kKeyBits) == 8u ? 1u : k & kKeyBits); }

// What choices go by, in 64 bits, of an expert with this logit and bias.
__device__ __forceinline__ double choice_score(const RouteArgs& p, float logit, float bias, const Row& row, double sum) {
  if (p.bias == nullptr) return logit;
  const double score = p.scoring == kSigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(logit)))
                       : row.broken          ? static_cast<double>(NAN)
                                             : exp(static_cast<double>(logit) - static_cast<double>(row.top)) / sum;
  return score + static_cast<double>(bias);
}

// The sum of a softmax.
template <int N>
__device__ __forceinline__ double sum_in_64_bits(const float (&logit)[N], const Row& row) {
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) sum += exp(static_cast<double>(logit[i]) - static_cast<double>(row.top));  // 0 where there is no expert
  return warp_sum(sum);
}

// The key of each lane's group in 64 bits, for groups of `span` lanes.
template <int N>
__device__ __noinline__ uint64_t group_in_64_bits(const RouteArgs& p, const float (&logit)[N], const Row& row, int lane, int span) {
  const bool sums = p.group_score == kTop2;
  const double sum = p.scoring == kSoftmax && p.bias != nullptr ? sum_in_64_bits<N>(logit, row) : 1.0;
  uint64_t first = 0, second = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = lane * N + i;
    const float bias = p.bias != nullptr && e < p.experts ? p.bias[e] : 0.0f;
    if (logit[i] == -INFINITY || bias == -INFINITY) continue;
    double v = choice_score(p, logit[i], bias, row, sum);
    if (sums && p.bias == nullptr)
      // a softmax's without its denominator, which is the same for all groups
      v = p.scoring == kSigmoid ? 1.0 / (1.0 + exp(-v)) : row.broken ? static_cast<double>(NAN) : exp(v - static_cast<double>(row.top));
    take(first, second, Order<double>::of(v));
  }
  for (int o = 1; o < span; o <<= 1) {
    const uint64_t b = __shfl_xor_sync(kFull, first, o), s = __shfl_xor_sync(kFull, second, o);
    take(first, second, b);
    take(first, second, s);
  }
  return group_key<double>(p.group_score, first, second);
}

// Whether this lane's group, of `span` lanes, is among the best.
template <class K>
__device__ __forceinline__ bool group_kept(const RouteArgs& p, K own, int lane, int span) {
  // the lanes of a group compare it with every span-th
  const int group = lane / span, mine = lane & (span - 1);
  int before = 0;  // groups that come before this lane's
  for (int g0 = 0; g0 < p.groups; g0 += span) {
    const int g = g0 + mine;
    const K other = __shfl_sync(kFull, own, g * span);
    before += g < p.groups && (other > own || (other == own && g < group));
  }
  for (int o = 1; o < span; o <<= 1) before += __shfl_xor_sync(kFull, before, o);
  return group < p.groups && before < p.top_groups;
}

// The first `count` experts in `chosen`, put in order in 64 bits. A lane has one.
template <int N>
__device__ __noinline__ void order_in_64_bits(const RouteArgs& p, const float (&logit)[N], float mine, const Row& row, int lane, uint16_t* chosen,
                                              int count) {
  const double sum = p.scoring == kSoftmax && p.bias != nullptr ? sum_in_64_bits<N>(logit, row) : 1.0;
  const int expert = lane < count ? chosen[lane] : 0;
  const float bias = p.bias != nullptr && lane < count ? p.bias[expert] : 0.0f;
  const uint64_t key = Order<double>::of(choice_score(p, mine, bias, row, sum));
  int before = 0;
  for (int i = 0; i < count; ++i) {
    const uint64_t other = __shfl_sync(kFull, key, i);
    const int e = __shfl_sync(kFull, expert, i);
    before += other > key || (other == key && e < expert);
  }
  __syncwarp();
  if (lane < count) chosen[before] = static_cast<uint16_t>(expert);
  __syncwarp();
}

// choose() for up to eight experts a lane, and groups that fill a power of two of lanes. `open`: not decided.
template <int DT, int N>
__device__ __forceinline__ int choose_quickly(const RouteArgs& p, int64_t token, const float (&logit)[N], const Row& row, int lane, Lists<N>& lists,
                                              bool& open) {
  constexpr bool kNarrow = DT != kF32;  // no bits are lost
  open = false;
  const int e0 = lane * N;
  uint32_t key[N];
  if (p.bias != nullptr) {
    float score[N], bias[N];
    load_values<kF32, N>(p.bias, e0, p.experts - e0, p.bias_vec != 0, bias);
    if (p.scoring == kSigmoid) {
#pragma unroll
      for (int i = 0; i < N; ++i) score[i] = quotient(1.0f, 1.0f + exp_of(-logit[i]));
    } else {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        score[i] = exp_of(logit[i] - row.top);  // 0 where there is no expert
        sum += score[i];
      }
      const float unit = row.broken ? NAN : quotient(1.0f, warp_sum(sum));
#pragma unroll
      for (int i = 0; i < N; ++i) score[i] *= unit;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = placed_key(score[i] + bias[i], i, logit[i] != -INFINITY && bias[i] != -INFINITY);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = placed_key(logit[i], i, logit[i] != -INFINITY);
  }
  sort_keys<N>(key);
  uint32_t best = key[0];  // this lane's largest
  const auto apart = [&](uint32_t upper, uint32_t lower) {  // certainly in this order
    if (upper == 0u || lower == 0u) return true;
    return p.bias != nullptr ? !near_by(upper == 8u ? 1u : upper, lower == 8u ? 1u : lower) : kNarrow || upper != lower;
  };

  if (p.groups > 1) {
    const int span = p.experts / p.groups / N;  // lanes of a group
    uint32_t first = key[0], second = N > 1 ? key[N > 1 ? 1 : 0] : 0u;
    const bool sums = p.group_score == kTop2;
    if (sums && p.bias == nullptr) {
      // of the two best logits; a softmax's without its denominator, which is the same for all groups
      first = second = 0u;
#pragma unroll
      for (int i = 0; i < N; ++i) take(first, second, logit[i] != -INFINITY ? Order<float>::of(logit[i]) : 0u);
      const auto score = [&](uint32_t k) {
        const float v = Order<float>::value(k);
        return k == 0u                ? 0u
               : p.scoring == kSigmoid ? Order<float>::of(quotient(1.0f, 1.0f + exp_of(-v)))
                                       : Order<float>::of(row.broken ? NAN : exp_of(v - row.top));
      };
      first = score(first);
      second = score(second);
    } else {
      first &= kKeyBits;
      second &= kKeyBits;
    }
    for (int o = 1; o < span; o <<= 1) {
      const uint32_t b = __shfl_xor_sync(kFull, first, o), s = __shfl_xor_sync(kFull, second, o);
      take(first, second, b);
      take(first, second, s);
    }
    uint32_t own = lane / span < p.groups ? first : 0u;
    float size = fabsf(key_value(first));
    if (sums && second != 0u) {
      own = Order<float>::of(key_value(first) + key_value(second));
      size += fabsf(key_value(second));
    }
    bool kept = group_kept(p, own, lane, span);
    if ((sums || p.bias != nullptr || !kNarrow) && p.top_groups < p.groups) {
      bool again;
      if (sums || p.bias != nullptr) {
        again = groups_near(own, kept, size);
      } else {
        const uint32_t lowest = __reduce_min_sync(kFull, kept ? own : 0xFFFFFFFFu);
        const uint32_t highest = __reduce_max_sync(kFull, kept ? 0u : own);
        again = lowest == highest && lowest != 0u;
      }
      if (again) kept = group_kept(p, group_in_64_bits<N>(p, logit, row, lane, span), lane, span);
    }
    if (!kept) best = 0u;
  }

#pragma unroll
  for (int i = 1; i < N; ++i) lists.key[i - 1][lane] = key[i];
  lists.key[N - 1][lane] = 0u;
  uint32_t mine = 0u;  // the key of this lane's choice
  int taken = 0;       // of this lane's list
  const auto choose_next = [&](int j, uint32_t largest) {
    if (lane == j) mine = largest;
    if (lane == __ffs(__ballot_sync(kFull, (best & kKeyBits) == largest)) - 1) {
      lists.chosen[j] = static_cast<uint16_t>(e0 + 7 - static_cast<int>(best & 7u));
      best = lists.key[taken++][lane];
    }
  };
  int count = 0;
  for (; count < p.top_k; ++count) {
    const uint32_t largest = __reduce_max_sync(kFull, best & kKeyBits);
    if (largest == 0u) break;
    choose_next(count, largest);
  }
  if (!kNarrow || p.bias != nullptr) {
    uint32_t next = __reduce_max_sync(kFull, best & kKeyBits);
    const uint32_t down = __shfl_down_sync(kFull, mine, 1), below = lane + 1 >= p.top_k ? next : down;
    if (__any_sync(kFull, lane < p.top_k && !apart(mine, below))) {
      // more experts, until one is certainly below: these are put in order
      uint32_t last = __shfl_sync(kFull, mine, p.top_k - 1);
      while (!apart(last, next) && count < 32) {
        choose_next(count++, next);
        last = next;
        next = __reduce_max_sync(kFull, best & kKeyBits);
      }
      open = !apart(last, next);
      __syncwarp();
      if (!open) {
        const float own = lane < count ? value_at<DT>(p.logits, token * p.stride + lists.chosen[lane]) : 0.0f;
        order_in_64_bits<N>(p, logit, own, row, lane, lists.chosen, count);
      }
    }
  }
  __syncwarp();
  const int chosen = lane < min(count, p.top_k) ? lists.chosen[lane] : -1;
  __syncwarp();  // before the next token's
  return chosen;
}

// A lane's share of a token's weights, before the scale: the score of its expert, renormalised or not.
struct Share {
  float score;  // of the expert
  float rest;   // 1 - score (sigmoid)
  float sum;    // what the score is divided by: of the token's scores, or 1
  bool floor;   // the sum is below 2^-100 and counts as that
};

constexpr float kLeast = 0x1p-100f;

// `logit`: of this lane's expert, if it has one. `total`: sum of all exp(logit - top) (softmax without renormalising).
__device__ __forceinline__ Share share_of(int scoring, bool renormalize, float logit, bool has, const Row& row, float total) {
  Share s{0.0f, 1.0f, 1.0f, false};
  if (scoring == kSigmoid) {
    if (has) {
      s.score = __fdiv_rn(1.0f, 1.0f + expf(-logit));
      s.rest = __fdiv_rn(1.0f, 1.0f + expf(logit));
    }
    if (renormalize) {
      s.sum = warp_sum(s.score);
      s.floor = s.sum < kLeast;
      if (s.floor) s.sum = kLeast;
    }
    return s;
  }
  if (renormalize) {
    // the scores' own denominator cancels: relative to the largest of the token's
    const uint32_t top = Order<float>::max_of(has ? Order<float>::of(logit) : 0u);
    if (has) s.score = expf(logit - Order<float>::value(top));
    s.sum = top == 0u ? 1.0f : warp_sum(s.score);
  } else {
    if (has) s.score = expf(logit - row.top);
    s.sum = total;
  }
  if (row.broken) s.score = NAN;
  return s;
}

template <int N>
__device__ __forceinline__ Row row_of(const float (&logit)[N]) {
  float all = logit[0], top = logit[0];  // a NaN if there is one; without NaNs
#pragma unroll
  for (int i = 1; i < N; ++i) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(all) : "f"(logit[i]));
    top = fmaxf(top, logit[i]);
  }
  Row row;
  row.broken = __any_sync(kFull, !(all < INFINITY));
  row.top = Order<float>::value(__reduce_max_sync(kFull, top == top ? Order<float>::of(top) : 0x007FFFFFu));
  if (row.top == -INFINITY) row.top = 0.0f;  // nothing is open
  return row;
}

// All of softmax's exponentials of a row, relative to its largest.
template <int N>
__device__ __forceinline__ float total_of(const float (&logit)[N], const Row& row) {
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) sum += expf(logit[i] - row.top);  // 0 where there is no expert
  return warp_sum(sum);
}

// --------------------------------------------------------------------- the order by expert
// The places of a block's choices, in the order of experts and within one of tokens. counts: choices of each chunk of
// tokens (chunks, pitch), 16-byte aligned, zeros behind the last expert. Shared: start (pitch + 32) words, parts
// (place_bytes of routing.cu). A thread adds up four experts over a share of the chunks, so that most loads of a share are in
// flight at once.
__device__ __forceinline__ void place(const RouteArgs& p, const int32_t* counts, int32_t* start, int32_t* parts) {
  const int threads = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quads = p.pitch >> 2, wide = min(threads, quads <= 32 ? 32 : 1 << (32 - __clz(quads - 1)));
  const int shares = threads / wide, share = threadIdx.x / wide, quad = threadIdx.x % wide;
  int4 total = make_int4(0, 0, 0, 0), before = total;
  if (quad < quads) {
    const int4* from = reinterpret_cast<const int4*>(counts) + quad;
    for (int c0 = share; c0 < p.chunks; c0 += 8 * shares) {
      int4 n[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = c0 + k * shares;
        n[k] = c < p.chunks ? from[static_cast<int64_t>(c) * quads] : make_int4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int has = c0 + k * shares < static_cast<int>(blockIdx.x) ? -1 : 0;
        total.x += n[k].x; total.y += n[k].y; total.z += n[k].z; total.w += n[k].w;
        before.x += n[k].x & has; before.y += n[k].y & has; before.z += n[k].z & has; before.w += n[k].w & has;
      }
    }
  }
  int4* totals = reinterpret_cast<int4*>(parts);
  totals[threadIdx.x] = total;
  totals[threads + threadIdx.x] = before;
  __syncthreads();
  // this chunk's first place within each expert: the experts' totals, scanned (wide * 4 of them, at most threads * 4)
  int32_t* warp_sums = start + p.pitch;
  int carry = 0;
  for (int e0 = 0; e0 < p.experts; e0 += threads) {
    const int e = e0 + threadIdx.x;
    int all = 0, mine = 0;
    if (e < p.experts)
      for (int k = 0; k < shares; ++k) {
        all += parts[k * wide * 4 + e];
        mine += parts[threads * 4 + k * wide * 4 + e];
      }
    int scan = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(kFull, scan, o);
      if (lane >= o) scan += up;
    }
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    int sums = lane < threads / 32 ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(kFull, sums, o);
      if (lane >= o) sums += up;
    }
    const int below = __shfl_sync(kFull, sums, (warp + 31) & 31), block_total = __shfl_sync(kFull, sums, 31);
    scan += carry + (warp == 0 ? 0 : below);
    if (e < p.experts) {
      start[e] = scan - all + mine;
      if (blockIdx.x == 0) p.ends[e] = scan;
    }
    carry += block_total;
    __syncthreads();
  }
  // places of no choice
  const int64_t places = p.tokens * p.top_k;
  for (int64_t i = carry + static_cast<int64_t>(blockIdx.x) * threads + threadIdx.x; i < places; i += static_cast<int64_t>(p.chunks) * threads)
    p.source[i] = -1;
  const int64_t from = static_cast<int64_t>(blockIdx.x) * p.chunk * p.top_k;
  const int items = static_cast<int>(min(static_cast<int64_t>(p.chunk) * p.top_k, places - from));
  // A warp takes 32 choices and leaves how many each expert has among them (table: warps x pitch, 16 bits); a thread an
  // expert then makes of the counts what the warps before have.
  uint16_t* table = reinterpret_cast<uint16_t*>(parts);
  for (int i0 = 0; i0 < items; i0 += threads) {
    const int warps = min(threads, items - i0 + 31) / 32;  // that have choices
    for (int i = threadIdx.x; i < warps * p.pitch / 2; i += threads) reinterpret_cast<uint32_t*>(table)[i] = 0u;
    __syncthreads();
    const int i = i0 + threadIdx.x;
    const int e = i < items ? p.experts_out[from + i] : -1;
    const uint32_t same = __match_any_sync(kFull, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && rank == 0) table[warp * p.pitch + e] = static_cast<uint16_t>(__popc(same));
    __syncthreads();
    for (int x = threadIdx.x; x < p.experts; x += threads) {
      int sum = 0;
#pragma unroll 8
      for (int w = 0; w < warps; ++w) {
        const int n = table[w * p.pitch + x];
        table[w * p.pitch + x] = static_cast<uint16_t>(sum);
        sum += n;
      }
      parts[warps * p.pitch / 2 + x] = sum;
    }
    __syncthreads();
    const int at = e >= 0 ? start[e] + table[warp * p.pitch + e] + rank : -1;
    if (i < items) p.rows[from + i] = at;
    if (at >= 0) p.source[at] = static_cast<int32_t>(from + i);
    __syncthreads();
    for (int x = threadIdx.x; x < p.experts; x += threads) start[x] += parts[warps * p.pitch / 2 + x];
  }
}

// A block has a chunk of tokens, its warps take them in turn. kOne: the one block of the call, which places its choices too.
template <int DT, int N, bool kOne>
__global__ void __launch_bounds__(N >= 16 ? 512 : 1024) route_kernel(const __grid_constant__ RouteArgs p) {
  extern __shared__ __align__(16) int32_t shared[];  // choices of each expert; kOne: and the starts
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  fp4::grid_launch_dependents();
  fp4::grid_wait();
  for (int e = threadIdx.x; e < p.pitch; e += blockDim.x) shared[e] = 0;
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.chunk, end = min(first + p.chunk, p.tokens);
  // the lists lie behind the counts, where choices are placed later
  auto& lists = reinterpret_cast<Lists<N>*>(shared + p.pitch)[warp];
  for (int64_t token = first + warp; token < end; token += warps) {
    int chosen = -1;
    float weight = 0.0f;
    if (p.mask == nullptr || p.mask[token] != 0) {
      float logit[N];
      load_values<DT, N>(p.logits, token * p.stride + lane * N, p.experts - lane * N, p.vec != 0, logit);
      const Row row = row_of<N>(logit);
      bool near, none;
      if constexpr (Lists<N>::kUsed) {
        if (p.quick != 0) chosen = choose_quickly<DT, N>(p, token, logit, row, lane, lists, near);
        else chosen = choose_apart<float, N>(p, logit, row, lane, near);
      } else {
        chosen = choose<float, N>(p, logit, row, lane, near);
      }
      if (near) chosen = choose_apart<double, N>(p, logit, row, lane, none);
      const float total = p.scoring == kSoftmax && p.renormalize == 0 ? total_of<N>(logit, row) : 1.0f;
      const float mine = chosen >= 0 ? value_at<DT>(p.logits, token * p.stride + chosen) : 0.0f;
      const Share s = share_of(p.scoring, p.renormalize != 0, mine, chosen >= 0, row, total);
      weight = chosen >= 0 ? __fdiv_rn(s.score, s.sum) * p.scale : 0.0f;
    }
    if (lane < p.top_k) {
      p.experts_out[token * p.top_k + lane] = chosen;
      p.weights[token * p.top_k + lane] = weight;
      if (chosen >= 0) atomicAdd(&shared[chosen], 1);  // a count, whatever the order
    }
  }
  __syncthreads();
  if constexpr (kOne) {
    place(p, shared, shared + p.pitch, shared + 2 * p.pitch + 32);  // over the lists, which are done with
  } else {
    for (int e = threadIdx.x; e < p.pitch; e += blockDim.x) p.counts[static_cast<int64_t>(blockIdx.x) * p.pitch + e] = shared[e];
  }
}

__global__ void __launch_bounds__(1024) place_kernel(const __grid_constant__ RouteArgs p) {
  extern __shared__ __align__(16) int32_t shared[];
  fp4::grid_launch_dependents();
  fp4::grid_wait();
  place(p, p.counts, shared, shared + p.pitch + 32);
}

// --------------------------------------------------------------------------- backward
struct RouteGradArgs {
  RouteArgs route;  // logits, experts_out and the rules
  const float* grad;
  void* dlogits;
};

template <int DT>
__device__ __forceinline__ void store_at(void* p, int64_t at, float v) {
  if constexpr (DT == kBF16) static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
  else if constexpr (DT == kF16) static_cast<__half*>(p)[at] = __float2half_rn(v);
  else static_cast<float*>(p)[at] = v;
}

// With the shares w of a token's weights and their gradients g (times the scale), S the sum that they were divided by:
// renormalised softmax: dl_j = w_j (g_j - sum g w), 0 for the others; softmax: dl_e = s_e ([e chosen] g - sum g s);
// sigmoid: dl_j = g_j s_j (1 - s_j), with (g_j - sum g w) / S in g_j's place where renormalised (g_j / 2^-100 where the
// sum is below that).
template <int DT, int N>
__global__ void __launch_bounds__(256) route_grad_kernel(const __grid_constant__ RouteGradArgs a) {
  const RouteArgs& p = a.route;
  const int lane = threadIdx.x & 31;
  fp4::grid_launch_dependents();
  fp4::grid_wait();
  const int64_t token = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  const int chosen = lane < p.top_k ? p.experts_out[token * p.top_k + lane] : -1;
  const bool has = chosen >= 0 && chosen < p.experts;
  const bool any = __any_sync(kFull, has);
  const bool whole = p.scoring == kSoftmax && any;  // the row itself is needed
  float logit[N];
  Row row{0.0f, false};
  float total = 1.0f;
  if (whole) {
    load_values<DT, N>(p.logits, token * p.stride + lane * N, p.experts - lane * N, p.vec != 0, logit);
    row = row_of<N>(logit);
    if (p.renormalize == 0) total = total_of<N>(logit, row);
  }
  const float mine = has ? value_at<DT>(p.logits, token * p.stride + chosen) : 0.0f;
  const Share s = share_of(p.scoring, p.renormalize != 0, mine, has, row, total);
  const float g = has ? a.grad[token * p.top_k + lane] * p.scale : 0.0f;
  const float w = __fdiv_rn(s.score, s.sum);
  const float mean = warp_sum(has ? g * w : 0.0f);
  float d;
  if (p.scoring == kSigmoid) {
    const float inner = p.renormalize == 0 ? g : __fdiv_rn(s.floor ? g : g - mean, s.sum);
    d = inner * s.score * s.rest;
  } else {
    d = w * (g - mean);
  }
  const bool others = whole && p.renormalize == 0;
  const int64_t at = token * p.experts;
  if (others) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane * N + i < p.experts)
        store_at<DT>(a.dlogits, at + lane * N + i, row.broken ? NAN : -__fdiv_rn(expf(logit[i] - row.top), total) * mean);
  } else {
    // zeros, in words where rows start on them
    constexpr int kEach = DT == kF32 ? 1 : 2;
    if ((p.experts % kEach) == 0 && (reinterpret_cast<uintptr_t>(a.dlogits) & 3) == 0) {
      uint32_t* words = static_cast<uint32_t*>(a.dlogits) + at / kEach;
      for (int i = lane; i < p.experts / kEach; i += 32) words[i] = 0u;
    } else {
      for (int e = lane; e < p.experts; e += 32) store_at<DT>(a.dlogits, at + e, 0.0f);
    }
  }
  __syncwarp();
  if (has) store_at<DT>(a.dlogits, at + chosen, d);
}

}  // namespace routing
