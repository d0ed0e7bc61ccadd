// routing.cu - host side and C ABI (include/piper_routing.h) of expert routing and the exchange of tokens.
#include "../../include/piper_routing.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <initializer_list>

#include "launch.cuh"
#include "routing_exchange.cuh"
#include "routing_route.cuh"

namespace {

// No std::string: nothing here throws across the C boundary.
thread_local char g_error[256];
std::atomic<uint64_t> g_launches{0};

int fail(int code, const char* message) {
  std::snprintf(g_error, sizeof(g_error), "%s", message);
  return code;
}

int cuda_fail(const char* what, cudaError_t e) {
  std::snprintf(g_error, sizeof(g_error), "%s: %s", what, cudaGetErrorString(e));
  return PIPER_ROUTING_ECUDA;
}

#define ROUTING_REQUIRE(condition, message) \
  if (!(condition)) return fail(PIPER_ROUTING_EINVAL, message)

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t width(int dtype) { return dtype == PIPER_ROUTING_F32 ? 4 : 2; }

int sm_count() {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> cached[kMaxDevices] = {};
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < kMaxDevices && (n = cached[dev].load(std::memory_order_relaxed)) > 0) return n;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  n = n > 0 ? n : 148;
  if (dev >= 0 && dev < kMaxDevices) cached[dev].store(n, std::memory_order_relaxed);
  return n;
}

cudaError_t launched() {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return cudaGetLastError();
}

template <class Args>
cudaError_t enqueue(void (*kernel)(Args), int64_t blocks, int threads, size_t smem, cudaStream_t stream, const Args& args) {
  cudaError_t e = cudaSuccess;
  // above 48 KB a kernel has to be allowed its shared memory: in every call all that a block can have, since another thread may
  // be between allowing it and its launch
  if (smem > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e == cudaSuccess) e = piper::launch(kernel, blocks, threads, smem, 1, stream, args);
  return e == cudaSuccess ? launched() : e;
}

int check_dtype(int dtype) {
  ROUTING_REQUIRE(dtype == PIPER_ROUTING_BF16 || dtype == PIPER_ROUTING_F16 || dtype == PIPER_ROUTING_F32,
                  "Routing supports bfloat16, float16 and float32 values.");
  return PIPER_ROUTING_OK;
}

int check_config(const piper_routing_config* c) {
  ROUTING_REQUIRE(c != nullptr, "Routing: null configuration.");
  ROUTING_REQUIRE(c->experts >= 1 && c->experts <= PIPER_ROUTING_MAX_EXPERTS, "Routing takes 1 to 1024 experts.");
  ROUTING_REQUIRE(c->top_k >= 1 && c->top_k <= PIPER_ROUTING_MAX_TOP_K && c->top_k <= c->experts,
                  "Routing: a token gets 1 to 32 experts, and no more than there are.");
  ROUTING_REQUIRE(c->tokens >= 0 && c->tokens < (int64_t{1} << 31) / c->top_k, "Routing: at most 2^31 choices.");
  ROUTING_REQUIRE(c->scoring == PIPER_ROUTING_SOFTMAX || c->scoring == PIPER_ROUTING_SIGMOID, "Routing: unknown scoring.");
  ROUTING_REQUIRE(c->groups >= 1 && c->groups <= PIPER_ROUTING_MAX_GROUPS && c->experts % c->groups == 0,
                  "Routing: 1 to 32 groups of equally many experts.");
  ROUTING_REQUIRE(c->top_groups >= 1 && c->top_groups <= c->groups, "Routing: a token's experts come from 1 to all groups.");
  ROUTING_REQUIRE(c->top_k <= c->experts / c->groups * c->top_groups, "Routing: a token's groups have fewer experts than it gets.");
  ROUTING_REQUIRE(c->group_score == PIPER_ROUTING_MAX || c->group_score == PIPER_ROUTING_TOP2, "Routing: unknown group score.");
  return PIPER_ROUTING_OK;
}

constexpr int64_t kOneBlockTokens = 128;

// Threads of a block that has the tokens of a chunk, a power of two: a warp a token, as many as registers for the experts of
// a lane leave.
int route_threads(int experts, int chunk) {
  int threads = 256;
  while (threads < chunk * 32 && threads < (experts > 256 ? 512 : 1024)) threads *= 2;
  return threads;
}

// A chunk of tokens for every SM, whole rounds of a block's warps where there are enough.
struct Chunks {
  int count, size;
};
Chunks chunks_of(const piper_routing_config& c) {
  if (c.tokens <= kOneBlockTokens) return {1, static_cast<int>(std::max<int64_t>(c.tokens, 1))};
  const int64_t size = std::max<int64_t>((c.tokens + sm_count() - 1) / sm_count(), 4);
  return {static_cast<int>((c.tokens + size - 1) / size), static_cast<int>(size)};
}

size_t counts_bytes(const piper_routing_config& c, const Chunks& n) {
  return n.count > 1 ? static_cast<size_t>(n.count) * ((c.experts + 3) / 4 * 4) * 4 : 0;
}

routing::RouteArgs route_args(const piper_routing_config& c) {
  routing::RouteArgs a{};
  a.tokens = c.tokens;
  a.experts = c.experts;
  a.pitch = (c.experts + 3) / 4 * 4;
  a.top_k = c.top_k;
  a.scoring = c.scoring;
  a.groups = c.groups;
  a.top_groups = c.top_groups;
  a.group_score = c.group_score;
  a.renormalize = c.renormalize != 0;
  a.scale = c.scale;
  return a;
}

#define ROUTING_TYPES(dtype, CALL)                                     \
  do {                                                                 \
    if ((dtype) == PIPER_ROUTING_BF16) { CALL(routing::kBF16); }       \
    else if ((dtype) == PIPER_ROUTING_F16) { CALL(routing::kF16); }    \
    else { CALL(routing::kF32); }                                      \
  } while (0)

// Whether a lane's N neighbouring values lie in pieces that one load takes, each there or not as a whole.
bool whole_pieces(const void* p, int64_t stride, int experts, int n, size_t size) {
  const size_t bytes = std::min<size_t>(16, n * size);
  return bytes >= 4 && aligned(p, bytes) && (stride * static_cast<int64_t>(size)) % static_cast<int64_t>(bytes) == 0 &&
         experts % static_cast<int>(bytes / size) == 0;
}

// Shared memory of placing choices: starts, and then in the same room sums of a thread's four experts or counts of each warp.
size_t place_bytes(int pitch, int threads) {
  return (pitch + 32 + std::max<size_t>(8 * threads, threads / 32 * static_cast<size_t>(pitch) / 2 + pitch)) * 4;
}

template <int DT, int N>
cudaError_t launch_route(routing::RouteArgs a, int threads, cudaStream_t s) {
  a.vec = whole_pieces(a.logits, a.stride, a.experts, N, width(DT));
  a.bias_vec = whole_pieces(a.bias, 0, a.experts, N, 4);
  const int span = a.experts / a.groups / N;
  a.quick = a.groups == 1 || (span > 0 && span * N * a.groups == a.experts && (span & (span - 1)) == 0);
  const size_t lists = threads / 32 * sizeof(routing::Lists<N>), places = place_bytes(a.pitch, threads);
  const auto kernel = a.chunks == 1 ? routing::route_kernel<DT, N, true> : routing::route_kernel<DT, N, false>;
  const size_t smem = a.pitch * 4 + (a.chunks == 1 ? std::max(lists, places) : lists);
  return enqueue(kernel, a.chunks, threads, smem, s, a);
}

template <int DT>
cudaError_t launch_route(const routing::RouteArgs& a, cudaStream_t s) {
  const int threads = route_threads(a.experts, a.chunk);
  if (a.experts <= 32) return launch_route<DT, 1>(a, threads, s);
  if (a.experts <= 64) return launch_route<DT, 2>(a, threads, s);
  if (a.experts <= 128) return launch_route<DT, 4>(a, threads, s);
  if (a.experts <= 256) return launch_route<DT, 8>(a, threads, s);
  if (a.experts <= 512) return launch_route<DT, 16>(a, threads, s);
  return launch_route<DT, 32>(a, threads, s);
}

template <int DT, int N>
cudaError_t launch_route_grad(routing::RouteGradArgs a, cudaStream_t s) {
  a.route.vec = whole_pieces(a.route.logits, a.route.stride, a.route.experts, N, width(DT));
  return enqueue(routing::route_grad_kernel<DT, N>, (a.route.tokens + 7) / 8, 256, 0, s, a);
}

template <int DT>
cudaError_t launch_route_grad(const routing::RouteGradArgs& a, cudaStream_t s) {
  const int n = a.route.experts;
  if (n <= 32) return launch_route_grad<DT, 1>(a, s);
  if (n <= 64) return launch_route_grad<DT, 2>(a, s);
  if (n <= 128) return launch_route_grad<DT, 4>(a, s);
  if (n <= 256) return launch_route_grad<DT, 8>(a, s);
  if (n <= 512) return launch_route_grad<DT, 16>(a, s);
  return launch_route_grad<DT, 32>(a, s);
}

int check_exchange(const piper_routing_exchange* e) {
  ROUTING_REQUIRE(e != nullptr, "Exchange: null description.");
  if (int rc = check_dtype(e->dtype)) return rc;
  ROUTING_REQUIRE(e->top_k >= 1 && e->top_k <= PIPER_ROUTING_MAX_TOP_K, "Exchange: a token has 1 to 32 choices.");
  ROUTING_REQUIRE(e->tokens >= 0 && e->tokens < (int64_t{1} << 31) / e->top_k, "Exchange: at most 2^31 choices.");
  ROUTING_REQUIRE(e->hidden >= 1 && e->hidden <= (1 << 24), "Exchange: tokens have 1 to 2^24 values.");
  ROUTING_REQUIRE(e->tokens == 0 || (e->rows != nullptr && e->total != nullptr), "Exchange: null rows or total.");
  return PIPER_ROUTING_OK;
}

// Values that a thread takes at once: 16 bytes' if every row of every tensor starts on such a boundary.
int values_at_once(const piper_routing_exchange& e, std::initializer_list<const void*> bases, std::initializer_list<int64_t> strides) {
  const int n = static_cast<int>(16 / width(e.dtype));
  for (const void* p : bases)
    if (!aligned(p, 16)) return 1;
  for (const int64_t s : strides)
    if (s % n != 0) return 1;
  return e.hidden % n == 0 ? n : 1;
}

// Choices whose rows a thread loads at once; with few it takes more pieces.
int choices_at_once(int top_k) { return top_k <= 2 ? 2 : top_k <= 4 ? 4 : 8; }

routing::ExchangeArgs exchange_args(const piper_routing_exchange& e, int values) {
  routing::ExchangeArgs a{};
  a.rows = e.rows;
  a.total = e.total;
  a.tokens = e.tokens;
  a.top_k = e.top_k;
  a.hidden = e.hidden;
  a.pieces = e.hidden / values;
  return a;
}

// V: 16 bytes' values, or one.
#define EXCHANGE_DISPATCH(dtype, wide, CALL)                               \
  do {                                                                     \
    if ((dtype) == PIPER_ROUTING_BF16) {                                   \
      if (wide) { CALL(routing::kBF16, 8); } else { CALL(routing::kBF16, 1); } \
    } else if ((dtype) == PIPER_ROUTING_F16) {                             \
      if (wide) { CALL(routing::kF16, 8); } else { CALL(routing::kF16, 1); }   \
    } else {                                                               \
      if (wide) { CALL(routing::kF32, 4); } else { CALL(routing::kF32, 1); }   \
    }                                                                      \
  } while (0)

}  // namespace

extern "C" {

int piper_routing_workspace(const piper_routing_config* c, size_t* bytes) {
  if (int rc = check_config(c)) return rc;
  ROUTING_REQUIRE(bytes != nullptr, "Routing: bad workspace query.");
  const Chunks n = chunks_of(*c);
  *bytes = counts_bytes(*c, n);
  return PIPER_ROUTING_OK;
}

int piper_routing_route(const piper_routing_config* c, const void* logits, int64_t stride, int32_t dtype,
                        const float* bias, const uint8_t* mask, float* weights, int32_t* experts, int32_t* ends,
                        int32_t* rows, int32_t* source, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_config(c)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  ROUTING_REQUIRE(ends != nullptr, "Routing: null ends.");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->tokens == 0) {
    const cudaError_t e = cudaMemsetAsync(ends, 0, sizeof(int32_t) * c->experts, s);
    return e == cudaSuccess ? PIPER_ROUTING_OK : cuda_fail("cudaMemsetAsync", e);
  }
  ROUTING_REQUIRE(logits != nullptr && weights != nullptr && experts != nullptr && rows != nullptr && source != nullptr,
                  "Routing: null input or output.");
  ROUTING_REQUIRE(aligned(logits, width(dtype)), "Routing: logits not aligned to their type.");
  ROUTING_REQUIRE(stride >= c->experts || c->tokens == 1, "Routing: rows of the logits overlap.");
  const Chunks n = chunks_of(*c);
  const size_t need = counts_bytes(*c, n);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(PIPER_ROUTING_EWORKSPACE, "Routing: workspace missing, too small or not aligned.");
  routing::RouteArgs a = route_args(*c);
  a.logits = logits;
  a.stride = stride;
  a.bias = bias;
  a.mask = mask;
  a.weights = weights;
  a.experts_out = experts;
  a.ends = ends;
  a.rows = rows;
  a.source = source;
  a.counts = static_cast<int32_t*>(workspace);
  a.chunk = n.size;
  a.chunks = n.count;
  cudaError_t e = cudaSuccess;
#define CALL(D) e = launch_route<D>(a, s)
  ROUTING_TYPES(dtype, CALL);
#undef CALL
  if (e != cudaSuccess) return cuda_fail("route kernel", e);
  if (n.count == 1) return PIPER_ROUTING_OK;
  e = enqueue(routing::place_kernel, n.count, 1024, place_bytes(a.pitch, 1024), s, a);
  return e == cudaSuccess ? PIPER_ROUTING_OK : cuda_fail("place kernel", e);
}

int piper_routing_route_grad(const piper_routing_config* c, const void* logits, int64_t stride, int32_t dtype,
                             const int32_t* experts, const float* grad, void* dlogits, void* stream) {
  if (int rc = check_config(c)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (c->tokens == 0) return PIPER_ROUTING_OK;
  ROUTING_REQUIRE(logits != nullptr && experts != nullptr && grad != nullptr && dlogits != nullptr, "Routing gradient: null input or output.");
  ROUTING_REQUIRE(aligned(logits, width(dtype)) && aligned(dlogits, width(dtype)), "Routing gradient: logits not aligned to their type.");
  ROUTING_REQUIRE(stride >= c->experts || c->tokens == 1, "Routing gradient: rows of the logits overlap.");
  routing::RouteGradArgs a{};
  a.route = route_args(*c);
  a.route.logits = logits;
  a.route.stride = stride;
  a.route.experts_out = const_cast<int32_t*>(experts);
  a.grad = grad;
  a.dlogits = dlogits;
  cudaError_t e = cudaSuccess;
#define CALL(D) e = launch_route_grad<D>(a, static_cast<cudaStream_t>(stream))
  ROUTING_TYPES(dtype, CALL);
#undef CALL
  return e == cudaSuccess ? PIPER_ROUTING_OK : cuda_fail("route gradient kernel", e);
}

int piper_routing_dispatch(const piper_routing_exchange* x, const void* in, int64_t in_stride, void* out, void* stream) {
  if (int rc = check_exchange(x)) return rc;
  if (x->tokens == 0) return PIPER_ROUTING_OK;
  ROUTING_REQUIRE(in != nullptr && out != nullptr, "Dispatch: null input or output.");
  ROUTING_REQUIRE(aligned(in, width(x->dtype)) && aligned(out, width(x->dtype)), "Dispatch: input or output not aligned to its type.");
  ROUTING_REQUIRE(in_stride >= 0, "Dispatch: negative stride.");
  const int values = values_at_once(*x, {in, out}, {in_stride});
  routing::ExchangeArgs a = exchange_args(*x, values);
  a.in = in;
  a.in_stride = in_stride;
  a.out = out;
  const int64_t blocks = (x->tokens * a.pieces + routing::kExchangeThreads - 1) / routing::kExchangeThreads;
  ROUTING_REQUIRE(blocks < (int64_t{1} << 31), "Dispatch: too many values for one call.");
  cudaError_t e = cudaSuccess;
#define CALL(D, V) e = enqueue(routing::dispatch_kernel<D, V>, blocks, routing::kExchangeThreads, 0, static_cast<cudaStream_t>(stream), a)
  EXCHANGE_DISPATCH(x->dtype, values > 1, CALL);
#undef CALL
  return e == cudaSuccess ? PIPER_ROUTING_OK : cuda_fail("dispatch kernel", e);
}

int piper_routing_combine(const piper_routing_exchange* x, const void* y, int64_t y_stride, const float* weights,
                          void* out, void* stream) {
  if (int rc = check_exchange(x)) return rc;
  if (x->tokens == 0) return PIPER_ROUTING_OK;
  ROUTING_REQUIRE(y != nullptr && out != nullptr, "Combine: null input or output.");
  ROUTING_REQUIRE(aligned(y, width(x->dtype)) && aligned(out, width(x->dtype)), "Combine: input or output not aligned to its type.");
  ROUTING_REQUIRE(y_stride >= 0, "Combine: negative stride.");
  const int values = values_at_once(*x, {y, out}, {y_stride});
  routing::ExchangeArgs a = exchange_args(*x, values);
  a.in = y;
  a.in_stride = y_stride;
  a.weights = weights;
  a.out = out;
  const int64_t each = routing::kExchangeThreads * (routing::kAtOnce / choices_at_once(x->top_k));
  const int64_t blocks = (x->tokens * a.pieces + each - 1) / each;
  ROUTING_REQUIRE(blocks < (int64_t{1} << 31), "Combine: too many values for one call.");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
#define CALL(D, V)                                                                                                       \
  e = choices_at_once(x->top_k) == 2   ? enqueue(routing::combine_kernel<D, V, 2>, blocks, routing::kExchangeThreads, 0, s, a) \
      : choices_at_once(x->top_k) == 4 ? enqueue(routing::combine_kernel<D, V, 4>, blocks, routing::kExchangeThreads, 0, s, a) \
                                       : enqueue(routing::combine_kernel<D, V, 8>, blocks, routing::kExchangeThreads, 0, s, a)
  EXCHANGE_DISPATCH(x->dtype, values > 1, CALL);
#undef CALL
  return e == cudaSuccess ? PIPER_ROUTING_OK : cuda_fail("combine kernel", e);
}

int piper_routing_combine_grad(const piper_routing_exchange* x, const void* y, int64_t y_stride, const float* weights,
                               const void* dout, int64_t dout_stride, void* dy, float* dweights, void* stream) {
  if (int rc = check_exchange(x)) return rc;
  if (x->tokens == 0) return PIPER_ROUTING_OK;
  ROUTING_REQUIRE(y != nullptr && weights != nullptr && dout != nullptr && dy != nullptr && dweights != nullptr,
                  "Combine gradient: null input or output.");
  ROUTING_REQUIRE(aligned(y, width(x->dtype)) && aligned(dout, width(x->dtype)) && aligned(dy, width(x->dtype)),
                  "Combine gradient: input or output not aligned to its type.");
  ROUTING_REQUIRE(y_stride >= 0 && dout_stride >= 0, "Combine gradient: negative stride.");
  const int values = values_at_once(*x, {y, dout, dy}, {y_stride, dout_stride});
  routing::ExchangeArgs a = exchange_args(*x, values);
  a.in = y;
  a.in_stride = y_stride;
  a.weights = weights;
  a.dout = dout;
  a.dout_stride = dout_stride;
  a.out = dy;
  a.dweights = dweights;
  const bool wide_blocks = x->tokens < 32 * sm_count();  // too few tokens to fill the SMs with a warp each
  const int64_t blocks = wide_blocks ? x->tokens : (x->tokens + 7) / 8;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
#define ENQUEUE(D, V, K)                                                                                               \
  (wide_blocks ? enqueue(routing::combine_grad_kernel<D, V, K, 8>, blocks, routing::kExchangeThreads, 0, s, a)          \
               : enqueue(routing::combine_grad_kernel<D, V, K, 1>, blocks, routing::kExchangeThreads, 0, s, a))
#define CALL(D, V) e = choices_at_once(x->top_k) == 2 ? ENQUEUE(D, V, 2) : choices_at_once(x->top_k) == 4 ? ENQUEUE(D, V, 4) : ENQUEUE(D, V, 8)
  EXCHANGE_DISPATCH(x->dtype, values > 1, CALL);
#undef CALL
#undef ENQUEUE
  return e == cudaSuccess ? PIPER_ROUTING_OK : cuda_fail("combine gradient kernel", e);
}

const char* piper_routing_last_error(void) { return g_error; }

const char* piper_routing_version(void) { return "piper-routing 0.1 sm_100a"; }

uint64_t piper_routing_launches(void) { return g_launches.load(std::memory_order_relaxed); }

}  // extern "C"
