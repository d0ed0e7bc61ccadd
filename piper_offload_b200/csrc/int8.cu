// int8.cu - host side and C ABI (include/piper_int8.h) of the 8-bit integer products.
#include "../../include/piper_int8.h"

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstdio>

#include "int8_few.cuh"
#include "int8_grad.cuh"
#include "int8_linear.cuh"
#include "int8_pair.cuh"
#include "int8_quant.cuh"
#include "launch.cuh"

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
  return PIPER_INT8_ECUDA;
}

#define INT8_REQUIRE(condition, message) \
  if (!(condition)) return fail(PIPER_INT8_EINVAL, message)

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    cudaGetLastError();
    return ok ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr) : nullptr;
  }();
  return fn;
}

// Encodes a 2-D map of 128-byte wide, 128-byte swizzled boxes. The encoder wants a current context, which a thread that has
// made no runtime call yet (autograd's own, for one) lacks: then the runtime makes its device's current first.
bool encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t cols, int64_t rows, int64_t pitch_bytes,
                int box_cols, int box_rows) {
  const auto enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch_bytes)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t one[2] = {1u, 1u};
  for (int attempt = 0; attempt < 2; ++attempt) {
    if (enc(map, type, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS)
      return true;
    if (cudaFree(nullptr) != cudaSuccess) return false;
  }
  return false;
}

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
int64_t align256(int64_t a) { return up(a, 256); }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t width(int dtype) { return dtype == PIPER_INT8_F32 ? 4 : 2; }

int check_dtype(int dtype) {
  INT8_REQUIRE(dtype == PIPER_INT8_BF16 || dtype == PIPER_INT8_F16 || dtype == PIPER_INT8_F32,
               "INT8 supports bfloat16, float16 and float32 values.");
  return PIPER_INT8_OK;
}

int check_matrix(const piper_int8_matrix* m) {
  INT8_REQUIRE(m != nullptr, "INT8: null matrix.");
  INT8_REQUIRE(m->batch > 0 && m->rows > 0 && m->cols > 0, "INT8 requires a non-empty matrix.");
  INT8_REQUIRE(m->cols <= PIPER_INT8_MAX_COLS, "INT8: at most 65536 columns, so that sums fit 32 bits.");
  INT8_REQUIRE(m->batch <= (int64_t{1} << 20) && m->rows < (int64_t{1} << 31) - 256 && m->batch * up(m->rows, 128) < (int64_t{1} << 31),
               "INT8: a matrix has at most 2^31 rows over its batch.");
  INT8_REQUIRE(m->scale_dtype >= 0 && m->scale_dtype <= 2, "INT8 scales are bfloat16, float16 or float32.");
  INT8_REQUIRE(m->per_row != 0 || m->batch == 1, "INT8: experts have a scale for each row.");
  return PIPER_INT8_OK;
}

int check_buffers(const piper_int8_matrix* m) {
  INT8_REQUIRE(m->codes != nullptr && m->scale != nullptr, "INT8: null codes or scales.");
  INT8_REQUIRE(aligned(m->scale, width(m->scale_dtype)), "INT8: scales are not aligned to their type.");
  return PIPER_INT8_OK;
}

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

i8::RowScales row_scales(const piper_int8_matrix& w) {
  return {w.scale, w.scale_dtype, w.per_row != 0 ? 1 : 0, w.over_127 != 0};
}

// Codes are used where they are if bulk copies can read them.
bool moves_codes(const piper_int8_matrix& w) { return w.cols % 16 != 0 || !aligned(w.codes, 16); }
int64_t code_pitch(const piper_int8_matrix& w) { return moves_codes(w) ? up(w.cols, 16) : w.cols; }

i8::RepackArgs repack_args(const piper_int8_matrix& w, uint8_t* out) {
  i8::RepackArgs r{};
  if (!moves_codes(w)) return r;
  r.codes = static_cast<const uint8_t*>(w.codes);
  r.out = out;
  r.cols = w.cols;
  r.pitch = code_pitch(w);
  r.pieces = w.batch * w.rows * (r.pitch / 16);
  return r;
}

// Warps that work on a row of `units` units: as few as hold it in their registers, `lane` units a lane, so that rows wait
// for few others; eight where there are too few rows for all SMs, or where rows have no whole units. bf16 to codes, four
// units a lane: 4096 x 4096 10.4 us with two warps, 14.3 with one or eight; x 8192 18.5 with four, 27.4 with one, 20.5 with
// eight; x 14336 30.8 with eight, 36.9 with four. bf16 gradients, two a lane while that is enough: 2048 x 4096 10.3 us with
// four warps, 12.3 with two or eight; x 8192 16.5 with eight, 20.0 with four; x 14336 31.9 with eight and four units, 34.4
// with two.
struct RowPlan {
  int warps;
  int64_t blocks;
  bool more;  // rows longer than two units a lane of eight warps
};
RowPlan plan_rows(int64_t rows, int64_t units, int64_t lane, bool vec) {
  int warps = 1;
  while (warps < 8 && units > 32 * lane * warps) warps *= 2;
  if (units > 64 && (rows < 8 * sm_count() || !vec)) warps = 8;
  if (!vec && units <= 64) warps = 1;
  return {warps, warps == 1 ? (rows + 7) / 8 : rows, units > 512};
}

// Rows that start on 16-byte boundaries and have whole units.
bool whole_units(const void* p, int64_t stride, int64_t rows, int64_t cols, int dtype) {
  return aligned(p, 16) && cols % i8::kUnit == 0 && (rows == 1 || (stride * static_cast<int64_t>(width(dtype))) % 16 == 0);
}

template <class Args, class Kernel>
cudaError_t launch_rows(int64_t blocks, cudaStream_t s, const RowPlan& rows, bool vec, const Args& args, const i8::RepackArgs& r, Kernel one, Kernel two,
                 Kernel four, Kernel eight, Kernel eight_more, Kernel one_any, Kernel eight_any) {
  const Kernel kernel = !vec              ? (rows.warps == 1 ? one_any : eight_any)
                        : rows.warps == 1 ? one
                        : rows.warps == 2 ? two
                        : rows.warps == 4 ? four
                        : rows.more       ? eight_more
                                          : eight;
  const cudaError_t e = piper::launch(kernel, blocks, i8::prepare_threads(rows.warps), 0, 1, s, args, r, static_cast<uint32_t>(rows.blocks));
  return e == cudaSuccess ? launched() : e;
}

int64_t repack_blocks(const i8::RepackArgs& r, const RowPlan& rows) {
  const int64_t threads = i8::prepare_threads(rows.warps);
  return (r.pieces + threads - 1) / threads;
}

// ---------------------------------------------------------------- the product
struct TilePlan {
  int bn, split;
  double cycles;
};

// Blocks of a cluster that share a tile's stages, by a rough account in cycles: a stage takes `stage`, leaving sums and
// adding them up 2500 and 80 for each token of the tile, and every wave of tiles 2000. Shared by four against not shared: 1 x
// 4096 x 4096 9.5 and 11.1 us, 24 tokens 9.9 and 11.2, 8 x 4096 x 14336 16.2 and 23.0, 128 x 4096 x 4096 in tiles of 128
// 14.6 and 14.1.
TilePlan plan_tile(int bn, int64_t items, int64_t stages, double stage, int64_t tile_tokens, bool can_split, int64_t room) {
  TilePlan best{bn, 1, 0.0};
  for (int split = 1; split <= (can_split ? i8::kMaxSplit : 1); split *= 2) {
    if (split > 1 && (items * split > room || stages < 2 * split)) break;
    const int64_t waves = (items * split + room - 1) / room;
    double cycles = static_cast<double>(waves) * (static_cast<double>((stages + split - 1) / split) * stage + 2000.0);
    if (split > 1) cycles += 2500.0 + 80.0 * static_cast<double>(tile_tokens);
    if (split == 1 || cycles < best.cycles) best = {bn, split, cycles};
  }
  return best;
}

// Token tiles to expect: of one weight's tokens, or of experts' that end inside their last tiles.
int64_t likely_tiles(int64_t batch, int64_t tokens, int64_t tile) {
  if (batch == 1) return (tokens + tile - 1) / tile;
  return std::max(std::min(batch, tokens), (tokens + tile * std::min(batch, tokens) / 2) / tile);
}

struct LinearPlan {
  int bn, split;
  bool pair;   // of SMs, on tiles of 256 outputs
  bool few;    // tokens, which the product quantises itself
  int x_stages, ring;  // of that: stages of a block, and how many are under way
  int blocks;  // on an SM
  int64_t x_pitch;
  int64_t x_codes, x_scale, x_sums, w_codes, total;  // byte offsets
};

// Whether two blocks share an SM, one starting or ending while the other streams: in small tiles, once there are more of them
// than SMs, and where blocks share sums (16 rows of 8 experts of 14336 x 4096 74.5 us, 76.6 with one block; 1024 rows of 32 of
// 2048 x 2048 31.4 and 35.4; 1 x 4096 x 4096 shared by four 9.5 and 10.1, but 24 x 4096 x 4096 not shared 11.7 and 11.2).
bool two_blocks(int bn, int64_t items, int split) { return bn <= 64 && (items > sm_count() || (bn == 32 && split > 1)); }

// A few tokens of one weight: one launch, if a block a tile, or a share of one, is enough and the tokens have so few values
// that every block can quantise them. One launch against two: 1 x 14336 x 4096 13.6 and 15.4 us, two tokens 13.7 and 15.5,
// four 16.0 and 15.5; 1 x 4096 x 4096 8.7 and 9.7; 8 x 1024 x 1024 5.8 and 6.3; 1 x 4096 x 14336 16.3 and 16.1. Clusters of
// eight blocks that fill their SMs find room for half of the SMs at most (1 x 2048 x 8192 shared by eight 13.9 us).
bool plan_few(const piper_int8_matrix& w, int64_t tokens, bool grouped, LinearPlan& plan) {
  const int64_t tiles = (w.rows + 127) / 128, stages = (w.cols + i8::kStageCols - 1) / i8::kStageCols;
  if (grouped || w.batch > 1 || tokens > i8::kFewTokens || tokens * w.cols > 8192 || moves_codes(w) || tiles > sm_count()) return false;
  int split = 1;
  while (split < 4 && tiles * split * 2 <= sm_count() && stages >= 8 * split) split *= 2;
  if (split == 4 && tiles * 16 <= sm_count() && stages >= 32) split = 8;
  const int64_t most = (stages + split - 1) / split;
  const int64_t ring = (i8::kSmemMax - 1024 - i8::few_smem(static_cast<int>(most), 0)) / i8::kFewStage;
  if (ring < 6) return false;
  LinearPlan p{};
  p.few = true;
  p.bn = i8::kFewTokens;
  p.blocks = 1;
  p.split = split;
  p.x_stages = static_cast<int>(most);
  p.ring = static_cast<int>(std::min<int64_t>(std::min<int64_t>(ring, i8::kFewRing), most));
  plan = p;
  return true;
}

LinearPlan plan_linear(const piper_int8_matrix& w, int64_t tokens, bool grouped) {
  LinearPlan p{};
  if (plan_few(w, tokens, grouped, p)) return p;
  const int64_t per_expert = (tokens + w.batch - 1) / w.batch;
  const int64_t stages = (w.cols + i8::kStageCols - 1) / i8::kStageCols;
  TilePlan best{};
  const auto items_of = [&](int bn, int64_t outputs) { return likely_tiles(w.batch, tokens, bn) * ((w.rows + outputs - 1) / outputs); };
  for (const int bn : {32, 64, 128, 256}) {
    // experts' weights stream from HBM: narrower tiles leave room for more of it under way (4096 rows of 32 experts of 2048 x
    // 2048 37.6 us in tiles of 128, 39.8 of 256)
    if (w.batch > 1 && bn == 256 && per_expert <= 192) break;
    const int64_t tile_tokens = std::min<int64_t>(up(per_expert, 16), bn), items = items_of(bn, 128);
    const int blocks = two_blocks(bn, items, 1) ? 2 : 1;
    const double stage = (300.0 + 2.0 * static_cast<double>(tile_tokens)) * (blocks == 2 ? 1.7 : 1.0);
    const TilePlan t = plan_tile(bn, items, stages, stage, tile_tokens, w.batch == 1 && blocks == 1, blocks * sm_count());
    if (best.bn == 0 || t.cycles < best.cycles) {
      best = t;
      p.blocks = two_blocks(bn, items, t.split) ? 2 : 1;
    }
  }
  // 4096 x 14336 x 4096 163 us on pairs, 184 on single SMs; 2048 x 4096 x 4096 34.0 and 35.0, 1024 23.9 and 23.5; 4096 rows
  // of 8 experts of 4096 x 2048 48.5 and 47.1
  for (const int bn : {128, 256}) {
    if (per_expert <= (w.batch == 1 ? 256 : 512)) break;
    const int64_t tile_tokens = std::min<int64_t>(up(per_expert, 32), bn);
    const TilePlan t = plan_tile(bn, items_of(bn, 256), stages, 290.0 + static_cast<double>(tile_tokens), tile_tokens, false, sm_count() / 2);
    if (t.cycles < best.cycles) {
      best = t;
      p.pair = true;
      p.blocks = 1;
    }
  }
  p.bn = best.bn;
  p.split = best.split;
  p.x_pitch = up(w.cols, 16);
  int64_t at = 0;
  p.x_codes = at;
  at += align256(tokens * p.x_pitch);
  p.x_scale = at;
  at += align256(tokens * 4);
  p.x_sums = at;
  if (w.zero != nullptr) at += align256(tokens * 4);
  p.w_codes = at;
  if (moves_codes(w)) at += align256(w.batch * w.rows * code_pitch(w));
  p.total = at;
  return p;
}

// Token tiles of all experts and of the rows after them (an upper bound: the ends are on the device), or of one weight's
// tokens (0 experts).
int64_t token_tiles(int64_t tokens, int64_t experts, int bn) {
  return experts == 0 ? (tokens + bn - 1) / bn : tokens / bn + std::min<int64_t>(experts + 1, tokens);
}

// A kernel's limit of shared memory is the same in every call, whatever the call takes: it is the kernel's, and another thread
// may be between setting it and its launch.
template <class Args>
cudaError_t launch(void (*kernel)(Args), const Args& args, int64_t blocks, int threads, int smem, int cluster, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, i8::kSmemMax);
  if (e != cudaSuccess) return e;
  e = piper::launch(kernel, blocks, threads, static_cast<size_t>(smem), cluster, stream, args);
  return e == cudaSuccess ? launched() : e;
}

template <int DT, int BN, int kCtas>
cudaError_t launch_linear(const i8::LinearArgs& args, int64_t items, cudaStream_t stream) {
  using S = i8::LinearShape<BN, kCtas>;
  return launch<i8::LinearArgs>(i8::linear_kernel<DT, BN, kCtas>, args, args.split > 1 ? items * args.split : std::min<int64_t>(items, kCtas * sm_count()),
                                i8::kLinearThreads, S::kSmem, args.split, stream);
}

template <int DT, int BN>
cudaError_t launch_pairs(const i8::LinearArgs& args, int64_t items, cudaStream_t stream) {
  return launch<i8::LinearArgs>(i8::linear_pair_kernel<DT, BN>, args, 2 * std::min<int64_t>(items, sm_count() / 2), i8::kLinearThreads,
                                i8::PairShape<BN>::kSmem, 2, stream);
}

int launch_few(const piper_int8_matrix& w, const LinearPlan& p, const void* x, int64_t x_stride, int64_t tokens, void* y, int dtype,
               cudaStream_t stream);

// --------------------------------------------------------------- the gradient
struct GradPlan {
  int terms;      // fp16 terms per value
  int64_t pitch;  // values between rows of terms
  int64_t values, back, w_codes, total;  // byte offsets
};

int grad_terms(int dtype) { return dtype == PIPER_INT8_F32 ? 2 : 1; }

GradPlan plan_grad(const piper_int8_matrix& w, int64_t tokens, int dtype) {
  GradPlan p{};
  p.terms = grad_terms(dtype);
  p.pitch = up(w.rows, i8::kUnit);
  int64_t at = 0;
  p.values = at;
  at += align256(p.terms * tokens * p.pitch * 2);
  p.back = at;
  at += align256(tokens * 4);
  p.w_codes = at;
  if (moves_codes(w)) at += align256(w.batch * w.rows * code_pitch(w));
  p.total = at;
  return p;
}

// Tiles of a gradient: tokens x columns. Decoding costs the same whatever the tokens, so tiles are as wide in tokens as they
// go, but for a few, which leave room for more stages. The rough account in cycles a stage was measured: one SM takes 810 for
// 128 columns x 256 tokens and 560 for few, a pair 1330 for 512 x 256 and 750 for 256 x 256 (2048 x 14336 x 4096 190 us in
// tiles of 512 on pairs, 200 of 256, on single SMs 233 of 128 x 256; 512 x 4096 x 4096 27 on single SMs that share sums, 30 on
// pairs; 512 rows of 16 experts of 2048 x 2048 27 in tiles of 512 on pairs, 30 of 128 x 64 on single SMs).
struct GradTile {
  int bn, rows, split;
  bool pair;
  int tokens;     // of a tile
  int64_t items;  // bound on the tiles
  int columns() const { return 128 * rows * (pair ? 2 : 1); }
};
GradTile grad_tile(const piper_int8_matrix& w, int64_t tokens, int terms, bool grouped) {
  const int64_t per_expert = std::max<int64_t>(tokens / w.batch, 1);
  const int64_t stages = (w.rows + i8::kGradStageRows - 1) / i8::kGradStageRows * terms;
  GradTile t{per_expert <= 48 ? 64 : 256, 1, 1, false, 0, 0};
  t.tokens = t.bn;
  const auto tiles = [&](int64_t columns, int64_t tile) { return likely_tiles(w.batch, tokens, tile) * ((w.cols + columns - 1) / columns); };
  const double one = std::max(560.0, 250.0 + 2.2 * static_cast<double>(std::min<int64_t>(per_expert, t.bn)));
  const TilePlan alone = plan_tile(t.bn, tiles(128, t.bn), stages, one, std::min<int64_t>(per_expert, t.bn), !grouped, sm_count());
  double best = alone.cycles;
  for (int rows = 1; rows <= 2; ++rows)
    // a stage of 192 tokens and fewer takes the same
    for (int tile = 256; tile >= 192; tile -= 32) {
      const double n = static_cast<double>(std::min<int64_t>(up(per_expert, 32), tile));
      const double stage = rows == 2 ? std::max(1000.0, 5.2 * n) : std::max(600.0, 2.95 * n);
      const int64_t room = sm_count() / 2, waves = (tiles(256 * rows, tile) + room - 1) / room;
      const double cycles = static_cast<double>(waves) * (static_cast<double>(stages) * stage + 2000.0);
      if (cycles < best) {
        best = cycles;
        t.pair = true;
        t.bn = 256;
        t.rows = rows;
        t.tokens = tile;
      }
    }
  t.items = token_tiles(tokens, grouped ? w.batch : 0, t.tokens) * ((w.cols + t.columns() - 1) / t.columns());
  // the account goes by even experts: there may be more tiles, which then are not shared
  if (!t.pair) t.split = plan_tile(t.bn, t.items, stages, one, std::min<int64_t>(tokens, t.bn), !grouped, sm_count()).split;
  return t;
}

template <int DT, int BN, int kRows, bool kPair>
cudaError_t launch_grad(const i8::GradArgs& args, int64_t items, cudaStream_t stream) {
  using S = i8::GradShape<BN, kRows, kPair>;
  static_assert(S::kCanSplit == !kPair, "the plan splits tiles that no pair has");
  const int cluster = kPair ? 2 : args.split;
  return launch<i8::GradArgs>(i8::grad_kernel<DT, BN, kRows, kPair>, args, items * cluster, S::kThreads, S::kSmem, cluster, stream);
}

#define INT8_DISPATCH(dtype, CALL)                              \
  do {                                                          \
    if ((dtype) == PIPER_INT8_BF16) { CALL(i8::kBF16); }        \
    else if ((dtype) == PIPER_INT8_F16) { CALL(i8::kF16); }     \
    else { CALL(i8::kF32); }                                    \
  } while (0)

template <int DT>
cudaError_t launch_few(const i8::FewArgs& args, int64_t tiles, cudaStream_t stream) {
  auto kernel = i8::linear_few_kernel<DT>;
  const int smem = i8::few_smem(args.x_stages, args.ring);
  return launch<i8::FewArgs>(kernel, args, tiles * args.split, i8::kFewThreads, smem, args.split, stream);
}

int launch_few(const piper_int8_matrix& w, const LinearPlan& p, const void* x, int64_t x_stride, int64_t tokens, void* y, int dtype,
               cudaStream_t stream) {
  i8::FewArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.rows_of = {row_scales(w), static_cast<const int8_t*>(w.zero), w.per_row != 0 ? 1 : 0};
  a.y = y;
  a.tokens = static_cast<int32_t>(tokens);
  a.rows = static_cast<int32_t>(w.rows);
  a.cols = static_cast<int32_t>(w.cols);
  a.split = p.split;
  a.x_stages = p.x_stages;
  a.ring = p.ring;
  a.vec = aligned(y, 16) && (w.rows * static_cast<int64_t>(width(dtype))) % 16 == 0;
  a.x_vec = whole_units(x, x_stride, tokens, w.cols, dtype);
  if (!encode_map(&a.w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, w.codes, w.cols, w.rows, w.cols, i8::kStageCols, fp4::kTileRows))
    return fail(PIPER_INT8_ECUDA, "INT8 product: cuTensorMapEncodeTiled failed.");
  const int64_t tiles = (w.rows + 127) / 128;
  cudaError_t e = cudaSuccess;
#define CALL(D) e = launch_few<D>(a, tiles, stream)
  INT8_DISPATCH(dtype, CALL);
#undef CALL
  return e == cudaSuccess ? PIPER_INT8_OK : cuda_fail("product kernel", e);
}

int check_call(const piper_int8_matrix* w, int64_t tokens, const int32_t* ends, int dtype) {
  if (int rc = check_matrix(w)) return rc;
  if (int rc = check_buffers(w)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  INT8_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 28), "INT8: too many tokens for one call.");
  INT8_REQUIRE(ends != nullptr || w->batch == 1, "INT8: several matrices need the ends of their rows.");
  return PIPER_INT8_OK;
}

}  // namespace

extern "C" {

int piper_int8_linear_workspace(const piper_int8_matrix* w, int64_t tokens, int32_t grouped, size_t* bytes) {
  if (int rc = check_matrix(w)) return rc;
  INT8_REQUIRE(bytes != nullptr && tokens >= 0 && (grouped != 0 || w->batch == 1), "INT8 product: bad workspace query.");
  *bytes = tokens == 0 ? 0 : static_cast<size_t>(plan_linear(*w, tokens, grouped != 0).total);
  return PIPER_INT8_OK;
}

int piper_int8_linear(const piper_int8_matrix* w, const void* x, int64_t x_stride, int64_t tokens, const int32_t* ends,
                      void* y, int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_call(w, tokens, ends, dtype)) return rc;
  if (tokens == 0) return PIPER_INT8_OK;
  INT8_REQUIRE(x != nullptr && y != nullptr, "INT8 product: null input or output.");
  INT8_REQUIRE(aligned(x, width(dtype)) && aligned(y, width(dtype)), "INT8 product: input or output not aligned to its type.");
  INT8_REQUIRE(x_stride >= w->cols || tokens == 1, "INT8 product: rows of the input overlap.");
  const LinearPlan p = plan_linear(*w, tokens, ends != nullptr);
  if (p.few) return launch_few(*w, p, x, x_stride, tokens, y, dtype, static_cast<cudaStream_t>(stream));
  if (workspace == nullptr || workspace_bytes < static_cast<size_t>(p.total) || !aligned(workspace, 256))
    return fail(PIPER_INT8_EWORKSPACE, "INT8 product: workspace missing, too small or not 256-byte aligned.");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);

  i8::QuantArgs q{};
  q.x = x;
  q.x_stride = x_stride;
  q.tokens = tokens;
  q.cols = static_cast<int32_t>(w->cols);
  q.pitch = p.x_pitch;
  q.codes = reinterpret_cast<int8_t*>(ws + p.x_codes);
  q.scale = reinterpret_cast<float*>(ws + p.x_scale);
  q.sums = w->zero != nullptr ? reinterpret_cast<int32_t*>(ws + p.x_sums) : nullptr;
  const i8::RepackArgs r = repack_args(*w, ws + p.w_codes);

  i8::LinearArgs a{};
  a.x_scale = q.scale;
  a.x_sums = q.sums;
  a.rows_of = {row_scales(*w), static_cast<const int8_t*>(w->zero), w->per_row != 0 ? 1 : 0};
  a.groups = {ends, tokens, static_cast<int32_t>(w->batch), static_cast<int32_t>(p.pair ? (w->rows + 255) / 256 : (w->rows + 127) / 128)};
  a.y = y;
  a.rows = static_cast<int32_t>(w->rows);
  a.cols = static_cast<int32_t>(w->cols);
  a.split = p.split;
  a.early = r.pieces == 0;
  a.vec = aligned(y, 16) && (w->rows * static_cast<int64_t>(width(dtype))) % 16 == 0;
  const int64_t items = token_tiles(tokens, ends == nullptr ? 0 : w->batch, p.bn) * a.groups.row_tiles;
  a.items = static_cast<int32_t>(items);
  INT8_REQUIRE(items < (int64_t{1} << 31) / i8::kMaxSplit, "INT8 product: too many tiles for one call.");
  const bool vec = whole_units(x, x_stride, tokens, w->cols, dtype);
  const RowPlan rows = plan_rows(tokens, p.x_pitch / i8::kUnit, dtype == PIPER_INT8_F32 ? 2 : 4, vec);
  const int64_t blocks = rows.blocks + repack_blocks(r, rows);
  INT8_REQUIRE(blocks < (int64_t{1} << 31), "INT8 product: too many values for one call.");
  const void* codes = r.pieces > 0 ? r.out : w->codes;
  if (!encode_map(&a.w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, w->cols, w->batch * w->rows, code_pitch(*w), i8::kStageCols, fp4::kTileRows) ||
      !encode_map(&a.x_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, q.codes, w->cols, tokens, p.x_pitch, i8::kStageCols, p.pair ? p.bn / 2 : p.bn))
    return fail(PIPER_INT8_ECUDA, "INT8 product: cuTensorMapEncodeTiled failed.");

  cudaError_t e = cudaSuccess;
#define CALL(D)                                                                                                              \
  constexpr int kHold = D == i8::kF32 ? 2 : 4;                                                                                \
  e = launch_rows(blocks, s, rows, vec, q, r, i8::quantize_kernel<D, 1, kHold, true>, i8::quantize_kernel<D, 2, kHold, true>,            \
              i8::quantize_kernel<D, 4, kHold, true>, i8::quantize_kernel<D, 8, 2, true>, i8::quantize_kernel<D, 8, kHold, true>,  \
              i8::quantize_kernel<D, 1, 2, false>,                                                                            \
              i8::quantize_kernel<D, 8, 2, false>)
  INT8_DISPATCH(dtype, CALL);
#undef CALL
  if (e != cudaSuccess) return cuda_fail("quantize kernel", e);
#define CALL(D)                                                                                                          \
  e = p.pair        ? (p.bn == 128 ? launch_pairs<D, 128>(a, items, s) : launch_pairs<D, 256>(a, items, s))                \
      : p.bn == 32  ? (p.blocks == 2 ? launch_linear<D, 32, 2>(a, items, s) : launch_linear<D, 32, 1>(a, items, s))        \
      : p.bn == 64  ? (p.blocks == 2 ? launch_linear<D, 64, 2>(a, items, s) : launch_linear<D, 64, 1>(a, items, s))        \
      : p.bn == 128 ? launch_linear<D, 128, 1>(a, items, s)                                                                \
                    : launch_linear<D, 256, 1>(a, items, s)
  INT8_DISPATCH(dtype, CALL);
#undef CALL
  return e == cudaSuccess ? PIPER_INT8_OK : cuda_fail("linear kernel", e);
}

int piper_int8_grad_input_workspace(const piper_int8_matrix* w, int64_t tokens, int32_t dtype, size_t* bytes) {
  if (int rc = check_matrix(w)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  INT8_REQUIRE(bytes != nullptr && tokens >= 0, "INT8 gradient: bad workspace query.");
  *bytes = tokens == 0 ? 0 : static_cast<size_t>(plan_grad(*w, tokens, dtype).total);
  return PIPER_INT8_OK;
}

int piper_int8_grad_input(const piper_int8_matrix* w, const void* dy, int64_t dy_stride, int64_t tokens,
                          const int32_t* ends, void* dx, int32_t dtype, void* workspace, size_t workspace_bytes,
                          void* stream) {
  if (int rc = check_call(w, tokens, ends, dtype)) return rc;
  if (tokens == 0) return PIPER_INT8_OK;
  INT8_REQUIRE(dy != nullptr && dx != nullptr, "INT8 gradient: null gradient or output.");
  INT8_REQUIRE(aligned(dy, width(dtype)) && aligned(dx, width(dtype)), "INT8 gradient: gradient or output not aligned to its type.");
  INT8_REQUIRE(dy_stride >= w->rows || tokens == 1, "INT8 gradient: rows of the gradient overlap.");
  const GradPlan p = plan_grad(*w, tokens, dtype);
  if (workspace == nullptr || workspace_bytes < static_cast<size_t>(p.total) || !aligned(workspace, 256))
    return fail(PIPER_INT8_EWORKSPACE, "INT8 gradient: workspace missing, too small or not 256-byte aligned.");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);

  i8::ScaleArgs v{};
  v.dy = dy;
  v.dy_stride = dy_stride;
  v.tokens = tokens;
  v.rows = static_cast<int32_t>(w->rows);
  v.pitch = p.pitch;
  v.out = reinterpret_cast<__half*>(ws + p.values);
  v.back = reinterpret_cast<float*>(ws + p.back);
  v.scales = row_scales(*w);
  v.ends = ends;
  v.experts = static_cast<int32_t>(w->batch);
  const i8::RepackArgs r = repack_args(*w, ws + p.w_codes);

  i8::GradArgs a{};
  const GradTile tile = grad_tile(*w, tokens, p.terms, ends != nullptr);
  a.codes = r.pieces > 0 ? r.out : static_cast<const uint8_t*>(w->codes);
  a.zero = static_cast<const int8_t*>(w->zero);
  a.back = v.back;
  a.groups = {ends, tokens, static_cast<int32_t>(w->batch), static_cast<int32_t>((w->cols + tile.columns() - 1) / tile.columns())};
  a.dx = dx;
  a.code_pitch = code_pitch(*w);
  a.zero_step = w->per_row != 0 ? 1 : 0;
  a.rows = static_cast<int32_t>(w->rows);
  a.cols = static_cast<int32_t>(w->cols);
  a.terms = p.terms;
  a.split = tile.split;
  a.tile_tokens = tile.tokens;
  a.vec = aligned(dx, 16) && (w->cols * static_cast<int64_t>(width(dtype))) % 16 == 0;
  const bool vec = whole_units(dy, dy_stride, tokens, w->rows, dtype) && aligned(w->scale, 16);
  const RowPlan rows = plan_rows(tokens, p.pitch / i8::kUnit, 2, vec);
  const int64_t blocks = rows.blocks + repack_blocks(r, rows);
  INT8_REQUIRE(tile.items < (int64_t{1} << 31) / i8::kMaxSplit && blocks < (int64_t{1} << 31), "INT8 gradient: too many tiles for one call.");
  if (!encode_map(&a.dy_map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, v.out, w->rows, p.terms * tokens, p.pitch * 2, i8::kGradStageRows, tile.pair ? tile.bn / 2 : tile.bn))
    return fail(PIPER_INT8_ECUDA, "INT8 gradient: cuTensorMapEncodeTiled failed.");

  cudaError_t e = cudaSuccess;
#define CALL(D)                                                                                                              \
  e = launch_rows(blocks, s, rows, vec, v, r, i8::scale_kernel<D, 1, 2, true>, i8::scale_kernel<D, 2, 2, true>, i8::scale_kernel<D, 4, 2, true>, \
              i8::scale_kernel<D, 8, 2, true>, i8::scale_kernel<D, 8, D == i8::kF32 ? 2 : 4, true>, i8::scale_kernel<D, 1, 2, false>,       \
              i8::scale_kernel<D, 8, 2, false>)
  INT8_DISPATCH(dtype, CALL);
#undef CALL
  if (e != cudaSuccess) return cuda_fail("scale kernel", e);
#define CALL(D)                                                                                              \
  e = tile.pair       ? (tile.rows == 2 ? launch_grad<D, 256, 2, true>(a, tile.items, s) : launch_grad<D, 256, 1, true>(a, tile.items, s)) \
      : tile.bn == 64 ? launch_grad<D, 64, 1, false>(a, tile.items, s)                                         \
                      : launch_grad<D, 256, 1, false>(a, tile.items, s)
  INT8_DISPATCH(dtype, CALL);
#undef CALL
  return e == cudaSuccess ? PIPER_INT8_OK : cuda_fail("gradient kernel", e);
}

int piper_int8_linear_plan(const piper_int8_matrix* w, int64_t tokens, int32_t grouped, piper_int8_plan* plan) {
  if (int rc = check_matrix(w)) return rc;
  INT8_REQUIRE(plan != nullptr && tokens > 0 && (grouped != 0 || w->batch == 1), "INT8 product: bad plan query.");
  const LinearPlan p = plan_linear(*w, tokens, grouped != 0);
  *plan = {p.bn, p.pair ? 256 : 128, p.split, p.blocks};
  return PIPER_INT8_OK;
}

int piper_int8_grad_input_plan(const piper_int8_matrix* w, int64_t tokens, int32_t grouped, int32_t dtype, piper_int8_plan* plan) {
  if (int rc = check_matrix(w)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  INT8_REQUIRE(plan != nullptr && tokens > 0 && (grouped != 0 || w->batch == 1), "INT8 gradient: bad plan query.");
  const GradTile t = grad_tile(*w, tokens, grad_terms(dtype), grouped != 0);
  *plan = {t.tokens, t.columns(), t.split, 1};
  return PIPER_INT8_OK;
}

const char* piper_int8_last_error(void) { return g_error; }

int piper_int8_device_status(void* stream, uint32_t* status) {
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail("cudaStreamSynchronize", e);
  unsigned int v = 0, zero = 0;
  e = cudaMemcpyFromSymbol(&v, pm::g_status, sizeof(v));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(pm::g_status, &zero, sizeof(zero));
  if (e != cudaSuccess) return cuda_fail("status word", e);
  if (status) *status = v;
  return v == 0 ? PIPER_INT8_OK : fail(PIPER_INT8_ETIMEOUT, "a bounded device-side wait timed out.");
}

const char* piper_int8_version(void) { return "piper-int8 0.1 sm_100a"; }

uint64_t piper_int8_launches(void) { return g_launches.load(std::memory_order_relaxed); }

}  // extern "C"
