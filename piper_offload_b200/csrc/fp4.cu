// fp4.cu - host side and C ABI (include/piper_fp4.h) of the FP4 operators.
#include "../../include/piper_fp4.h"

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstdio>

#include "fp4_grad.cuh"
#include "fp4_linear.cuh"
#include "fp4_quant.cuh"

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
  return PIPER_FP4_ECUDA;
}

#define FP4_REQUIRE(condition, message) \
  if (!(condition)) return fail(PIPER_FP4_EINVAL, message)

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

// Encodes a 2-D map of 128-byte wide, 128-byte swizzled boxes. The encoder wants
// a current context, which a thread that has made no runtime call yet (autograd's
// own, for one) lacks: then the runtime makes its device's current first.
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

int block_of(const piper_fp4_matrix& m) { return m.format == PIPER_FP4_MX ? 32 : 16; }
size_t width(int dtype) { return dtype == PIPER_FP4_BF16 ? 2 : 4; }

int check_matrix(const piper_fp4_matrix* m) {
  FP4_REQUIRE(m != nullptr, "FP4: null matrix.");
  FP4_REQUIRE(m->format == PIPER_FP4_MX || m->format == PIPER_FP4_NV, "FP4: unknown format.");
  FP4_REQUIRE(m->batch > 0 && m->rows > 0 && m->cols > 0, "FP4 requires a non-empty matrix.");
  FP4_REQUIRE(m->cols % block_of(*m) == 0,
              m->format == PIPER_FP4_MX ? "MXFP4 requires columns divisible by 32." : "NVFP4 requires columns divisible by 16.");
  FP4_REQUIRE(m->batch <= (int64_t{1} << 20) && m->rows < (int64_t{1} << 31) - 256 && m->cols < (int64_t{1} << 31) - 256 &&
                  m->batch * up(m->rows, 128) < (int64_t{1} << 31),
              "FP4: a matrix has at most 2^31 rows over its batch and 2^31 columns.");
  FP4_REQUIRE(m->format == PIPER_FP4_NV || m->second == nullptr, "MXFP4 has no second-level scale.");
  return PIPER_FP4_OK;
}

int check_buffers(const piper_fp4_matrix* m) {
  FP4_REQUIRE(m->codes != nullptr && m->scale != nullptr, "FP4: null codes or scales.");
  return PIPER_FP4_OK;
}

int check_dtype(int dtype) {
  FP4_REQUIRE(dtype == PIPER_FP4_BF16 || dtype == PIPER_FP4_F32, "FP4 supports bfloat16 and float32 values.");
  return PIPER_FP4_OK;
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

// Scales per row (row-major) or scale tiles per row (swizzled).
int scale_cols(const piper_fp4_matrix& m) {
  const int64_t blocks = m.cols / block_of(m);
  return static_cast<int>(m.swizzled ? (blocks + 3) / 4 : blocks);
}

// Rows that a lane quantizes: several, whose loads are in flight together, once there are blocks for every SM;
// before that one, as a lane's rows come one after another (24 x 4096: 2.3 us with 1, 3.6 with 4).
int many_rows(int dtype) { return dtype == PIPER_FP4_BF16 ? fp4::quant_rows<fp4::kBF16>() : fp4::quant_rows<fp4::kF32>(); }
int rows_per_lane(const fp4::QuantArgs& q, int dtype) {
  return fp4::quant_blocks(q, many_rows(dtype)) < 2 * sm_count() ? 1 : many_rows(dtype);
}

#define FP4_DISPATCH(dtype, format, CALL)                          \
  do {                                                             \
    if ((dtype) == PIPER_FP4_BF16) {                               \
      if ((format) == PIPER_FP4_MX) { CALL(fp4::kBF16, fp4::kMX); } \
      else { CALL(fp4::kBF16, fp4::kNV); }                         \
    } else {                                                       \
      if ((format) == PIPER_FP4_MX) { CALL(fp4::kF32, fp4::kMX); } \
      else { CALL(fp4::kF32, fp4::kNV); }                          \
    }                                                              \
  } while (0)

// ---------------------------------------------------------------- the product
// How a product runs, and its scratch: quantized tokens, and codes that are
// not stored as the product reads them.
struct LinearPlan {
  bool fused;       // tokens are quantized by the product itself
  bool move_codes;
  int bn, split;    // tokens per tile, blocks per tile
  int64_t k_padded; // columns up to a whole scale tile
  int64_t x_codes, x_scale, w_codes, total;  // byte offsets
  int64_t w_code_pitch, scale_tiles, scale_rows;
};

// Tokens per tile and blocks of a cluster that share a tile's stages, by a
// rough account in cycles: a stage takes `stage`, leaving sums and adding them
// up 2500 and 30 for each token of the tile, and every wave of tiles 2000.
// Split against not: 1 x 4096 x 14336 NVFP4 10.7 and 19.1 us, 24 x 4096 x 4096 MXFP4
// 9.0 and 10.5, 128 x 4096 x 14336 NVFP4 15.5 and 19.3. `room` is how many blocks
// the GPU holds; with two on an SM fewer than four stages a block do not pay (1 x
// 4096 x 4096 MXFP4 split in 8 8.2 us, in 4 6.1).
struct TilePlan {
  int bn, split;
  double cycles;
};
TilePlan plan_tile(int bn, int64_t items, int64_t stages, double stage, int64_t tile_tokens, bool can_split, int64_t room) {
  TilePlan best{bn, 1, 0.0};
  for (int split = 1; split <= (can_split ? fp4::kMaxSplit : 1); split *= 2) {
    if (split > 1 && (items * split > room || stages < (room > sm_count() ? 4 : 2) * split)) break;
    const int64_t waves = (items * split + room - 1) / room;
    double cycles = static_cast<double>(waves) * (static_cast<double>((stages + split - 1) / split) * stage + 2000.0);
    if (split > 1) cycles += 2500.0 + 30.0 * static_cast<double>(tile_tokens);
    if (split == 1 || cycles < best.cycles) best = {bn, split, cycles};
  }
  return best;
}

LinearPlan plan_linear(const piper_fp4_matrix& w, int64_t tokens) {
  LinearPlan p{};
  const int64_t per_expert = (tokens + w.batch - 1) / w.batch;
  // One or two tokens a weight, and few enough tiles that no block quantizes them again for another: one launch less
  // (5.8 us of host time against 8.6). On the device, fused against prepared: 1 x 14336 x 4096 NVFP4 9.6 and 10.0 us,
  // 1 x 28672 x 4096 14.5 and 17.5, 2 x 4096 x 4096 MXFP4 6.2 and 7.3, 8 rows over 8 experts of 2816 x 1024 6.3 and 8.0.
  // A block quantizes two tokens of a stage at a time, so the product of both is bounded in case one expert has all the
  // rows (128 over 64 experts of 512 x 1024 NVFP4, fused without that bound: 8.0 us evenly, 13.1 with most in one;
  // prepared 8.4 and 7.3).
  const int64_t stages = (w.cols + fp4::kStageCols - 1) / fp4::kStageCols;
  p.fused = tokens / w.batch <= 2 && std::min(w.batch, tokens) * ((w.rows + 127) / 128) <= fp4::kFusedCtas * sm_count() &&
            (w.batch == 1 || tokens * stages <= 128);
  // 333 tokens x 1000 x 2080 MXFP4: 10.1 us in tiles of 32, 12.2 of 192; 512 x 4096 x 14336 NVFP4: 24.7 of 128, 32.9 of
  // 192; 4096 x 14336 x 4224: 145.5 of 128, 141 of 192
  TilePlan best{};
  for (const int bn : {32, 128, 192}) {
    if (p.fused && bn > 32) break;
    const int64_t tile_tokens = std::min<int64_t>(up(per_expert, 16), bn);
    const int64_t items = std::min(w.batch, tokens) * ((per_expert + bn - 1) / bn) * ((w.rows + 127) / 128);
    const TilePlan t = plan_tile(bn, items, stages,
                                 330.0 + 2.0 * static_cast<double>(tile_tokens), tile_tokens, w.batch == 1, (p.fused ? fp4::kFusedCtas : 1) * sm_count());
    if (best.bn == 0 || t.cycles < best.cycles) best = t;
  }
  p.bn = best.bn;
  p.split = best.split;
  const int tile = block_of(w) * 4;
  p.scale_tiles = (w.cols + tile - 1) / tile;
  p.k_padded = p.scale_tiles * tile;
  p.move_codes = w.cols % 32 != 0 || !aligned(w.codes, 16);
  p.w_code_pitch = up(w.cols / 2, 16);
  int64_t at = 0;
  if (!p.fused) {
    // one more than first_scale_row's numbers can reach
    p.scale_rows = (tokens / p.bn + w.batch + 1) * fp4::scale_rows_per_tile(p.bn);
    p.x_codes = at;
    at += align256(tokens * (p.k_padded / 2));
    p.x_scale = at;
    at += align256(p.scale_rows * p.scale_tiles * 4);
  }
  p.w_codes = at;
  if (p.move_codes) at += align256(w.batch * w.rows * p.w_code_pitch);
  p.total = at;
  return p;
}

// Map of rows of packed codes, in boxes of 256 values x `box_rows` rows with the 128-byte swizzle.
bool code_map(CUtensorMap* map, const void* base, int64_t row_bytes, int64_t pitch, int64_t rows, int box_rows) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, row_bytes, rows, pitch, fp4::kStageBytes, box_rows);
}

// Token tiles of all experts and of the rows after them (an upper bound: the ends are on the device), or of one
// weight's tokens (0 experts).
int64_t token_tiles(int64_t tokens, int64_t experts, int bn) {
  return experts == 0 ? (tokens + bn - 1) / bn : tokens / bn + std::min<int64_t>(experts + 1, tokens);
}

template <int DT, int FMT, int BN, bool kFused>
cudaError_t launch_linear(fp4::LinearArgs& args, int64_t items, cudaStream_t stream) {
  using S = fp4::LinearShape<FMT, BN, kFused>;
  auto kernel = fp4::linear_kernel<DT, FMT, BN, kFused>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  static_assert(S::kCanSplit, "the plan may split any tile");
  cudaLaunchAttribute attributes[2] = {};
  // may start while the launch before it still quantizes; the kernel waits where it needs that
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = kFused ? 0 : 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = static_cast<unsigned>(args.split);
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(
      args.split > 1 ? items * args.split : std::min<int64_t>(items, S::kCtas * sm_count())));
  config.blockDim = dim3(S::kThreads);
  config.dynamicSmemBytes = S::kSmem;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = args.split > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&config, kernel, args);
  return e == cudaSuccess ? launched() : e;
}

// --------------------------------------------------------------- the gradient
struct GradPlan {
  bool move;      // dy goes through the workspace
  int terms;      // bf16 terms per value
  int64_t pitch;  // values between its rows there
  int64_t total;  // bytes
};

int grad_terms(int dtype) { return dtype == PIPER_FP4_F32 ? 3 : 1; }

GradPlan plan_grad(const piper_fp4_matrix& w, const void* dy, int64_t stride, int64_t tokens, int dtype) {
  GradPlan p{};
  p.terms = grad_terms(dtype);
  p.move = p.terms > 1 || !aligned(dy, 16) || (stride % 8 != 0 && tokens > 1);
  p.pitch = up(w.rows, 8);
  p.total = p.move ? align256(p.terms * tokens * p.pitch * 2) : 0;
  return p;
}

// Tiles of a gradient: tokens x (rows x 128) columns. Decoding costs the same
// whatever the tokens, so tiles are as wide in tokens as they go, but for a few,
// which leave room for more stages (32 x 14336 x 4096 NVFP4: 31.1 us in tiles of 64,
// 36.6 of 256); 256 columns where that fills the SMs (a rough account in cycles a
// stage: 1060 and 600; 2048 x 14336 x 4096 198 us against 231 with 128 columns,
// 512 x 4096 x 4096 60 against 25.8).
struct GradTile {
  int bn, rows, split;
  int64_t items;  // bound on the tiles
};
GradTile grad_tile(const piper_fp4_matrix& w, int64_t tokens, int terms, bool grouped) {
  const int64_t per_expert = tokens / w.batch;
  GradTile t{256, 1, 1, 0};
  if (per_expert <= 48) {
    t.bn = 64;
  } else {
    const auto waves = [&](int64_t cols) {
      const int64_t tiles = w.batch * ((per_expert + 255) / 256) * ((w.cols + cols - 1) / cols);
      return static_cast<double>((tiles + sm_count() - 1) / sm_count());
    };
    if (waves(256) * 1060.0 <= waves(128) * 600.0) t.rows = 2;
  }
  t.items = token_tiles(tokens, grouped ? w.batch : 0, t.bn) * ((w.cols + 128 * t.rows - 1) / (128 * t.rows));
  const int64_t stages = (w.rows + fp4::kGradStageRows - 1) / fp4::kGradStageRows * terms;
  t.split = plan_tile(t.bn, t.items, stages, 600.0, std::min<int64_t>(tokens, t.bn), t.rows == 1 && !grouped, sm_count()).split;
  return t;
}

template <int DT, int FMT, int BN, int kRows>
cudaError_t launch_grad(const fp4::GradArgs& args, int64_t items, cudaStream_t stream) {
  using S = fp4::GradShape<BN, kRows>;
  static_assert(S::kCanSplit == (kRows == 1), "the plan splits tiles of 128 columns");
  auto kernel = fp4::grad_kernel<DT, FMT, BN, kRows>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = static_cast<unsigned>(args.split);
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(items * args.split));
  config.blockDim = dim3(S::kThreads);
  config.dynamicSmemBytes = S::kSmem;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = args.split > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&config, kernel, args);
  return e == cudaSuccess ? launched() : e;
}

}  // namespace

extern "C" {

int piper_fp4_quantize(const piper_fp4_matrix* m, const void* x, int64_t x_stride, int32_t dtype, int32_t scale_mode,
                       int32_t second_mode, uint32_t* maxima, void* stream) {
  if (int rc = check_matrix(m)) return rc;
  if (int rc = check_buffers(m)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  FP4_REQUIRE(x != nullptr, "FP4 quantisation: null input.");
  FP4_REQUIRE(x_stride >= m->cols || (m->rows == 1 && m->batch == 1), "FP4 quantisation: rows of the input overlap.");
  FP4_REQUIRE(scale_mode >= 0 && scale_mode <= 3, "Unsupported MX scaling mode id.");
  FP4_REQUIRE(second_mode >= 0 && second_mode <= 2, "FP4 quantisation: unknown second-level mode.");
  FP4_REQUIRE((second_mode == PIPER_FP4_SECOND_NONE) == (m->second == nullptr),
              "FP4 quantisation: the second-level scale does not match its mode.");
  FP4_REQUIRE(aligned(m->codes, 4) && (!m->swizzled || aligned(m->scale, 4)),
              "FP4 quantisation: codes and swizzled scales start on 4-byte boundaries.");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int tile = block_of(*m) * 4;
  fp4::QuantArgs q{};
  q.x = x;
  q.x_stride = x_stride;
  q.rows = m->rows;
  q.rows_padded = m->swizzled ? up(m->rows, 128) : m->rows;
  q.batch = m->batch;
  q.cols = static_cast<int32_t>(m->cols);
  q.units = static_cast<int32_t>((m->swizzled ? up(m->cols, tile) : m->cols) / fp4::kUnit);
  q.vec = aligned(x, 32) && (x_stride * static_cast<int64_t>(width(dtype))) % 32 == 0;
  q.pairs = aligned(m->codes, 8);
  q.codes = static_cast<uint8_t*>(m->codes);
  q.code_pitch = m->cols / 2;
  q.scale = static_cast<uint8_t*>(m->scale);
  q.scale_cols = scale_cols(*m);
  q.swizzled = m->swizzled != 0;
  q.words = m->cols % tile == 0 || m->swizzled ? aligned(m->scale, 4) : 0;
  q.scale_mode = scale_mode;
  q.second_mode = second_mode;
  q.second = m->second;
  if (second_mode == PIPER_FP4_SECOND_COMPUTE) {
    FP4_REQUIRE(m->batch <= 65535, "FP4 quantisation: at most 65535 matrices with second-level scales.");
    q.reverse = 1;
    // one launch of one block a matrix instead of a clear, a maximum and a quantisation: 70 x 208 in 5.5 us against 10
    if (m->rows * m->cols <= PIPER_FP4_SMALL_MATRIX) {
#define CALL(D, F) fp4::quantize_small_kernel<D, F><<<static_cast<unsigned>(m->batch), fp4::kSmallThreads, 0, s>>>(q)
      FP4_DISPATCH(dtype, m->format, CALL);
#undef CALL
      const cudaError_t e = launched();
      return e == cudaSuccess ? PIPER_FP4_OK : cuda_fail("quantize kernel", e);
    }
    FP4_REQUIRE(maxima != nullptr, "FP4 quantisation: computing second-level scales needs room for the maxima.");
    q.amax = maxima;
    cudaError_t e = cudaMemsetAsync(maxima, 0, sizeof(uint32_t) * m->batch, s);
    if (e != cudaSuccess) return cuda_fail("cudaMemsetAsync", e);
    const int64_t blocks = fp4::quant_row_blocks(q, many_rows(dtype)) * ((q.units + 31) / 32);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, int64_t{32} * sm_count())), static_cast<unsigned>(m->batch));
    if (dtype == PIPER_FP4_BF16) fp4::amax_kernel<fp4::kBF16><<<grid, fp4::kQuantThreads, 0, s>>>(q, maxima);
    else fp4::amax_kernel<fp4::kF32><<<grid, fp4::kQuantThreads, 0, s>>>(q, maxima);
    if ((e = launched()) != cudaSuccess) return cuda_fail("amax kernel", e);
  }
  const int lane_rows = rows_per_lane(q, dtype);
  q.row_blocks = static_cast<int32_t>(fp4::quant_row_blocks(q, lane_rows));
  const int64_t blocks = fp4::quant_blocks(q, lane_rows);
  FP4_REQUIRE(blocks < (int64_t{1} << 31), "FP4 quantisation: too many values for one call.");
#define CALL(D, F)                                                                                                \
  if (lane_rows == 1) fp4::quantize_kernel<D, F, 1><<<static_cast<unsigned>(blocks), fp4::kQuantThreads, 0, s>>>(q); \
  else fp4::quantize_kernel<D, F, fp4::quant_rows<D>()><<<static_cast<unsigned>(blocks), fp4::kQuantThreads, 0, s>>>(q)
  FP4_DISPATCH(dtype, m->format, CALL);
#undef CALL
  const cudaError_t e = launched();
  return e == cudaSuccess ? PIPER_FP4_OK : cuda_fail("quantize kernel", e);
}

int piper_fp4_dequantize(const piper_fp4_matrix* m, void* y, int32_t dtype, void* stream) {
  if (int rc = check_matrix(m)) return rc;
  if (int rc = check_buffers(m)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  FP4_REQUIRE(y != nullptr, "FP4 dequantisation: null output.");
  fp4::DequantArgs d{};
  d.codes = static_cast<const uint8_t*>(m->codes);
  d.scale = static_cast<const uint8_t*>(m->scale);
  d.second = m->second;
  d.y = y;
  d.rows = m->rows;
  d.batch = m->batch;
  d.cols = static_cast<int32_t>(m->cols);
  d.swizzled = m->swizzled != 0;
  d.scale_cols = scale_cols(*m);
  d.vec = aligned(m->codes, 8) && aligned(y, 32);
  const int units = d.cols / fp4::kUnit;
  const int64_t block_rows = fp4::kQuantThreads / fp4::lanes_per_row(units) * fp4::kDequantRows;
  const int64_t blocks = m->batch * ((m->rows + block_rows - 1) / block_rows) * ((units + 31) / 32);
  FP4_REQUIRE(blocks < (int64_t{1} << 31), "FP4 dequantisation: too many values for one call.");
#define CALL(D, F) \
  fp4::dequantize_kernel<D, F><<<static_cast<unsigned>(blocks), fp4::kQuantThreads, 0, static_cast<cudaStream_t>(stream)>>>(d)
  FP4_DISPATCH(dtype, m->format, CALL);
#undef CALL
  const cudaError_t e = launched();
  return e == cudaSuccess ? PIPER_FP4_OK : cuda_fail("dequantize kernel", e);
}

int piper_fp4_linear_workspace(const piper_fp4_matrix* w, int64_t tokens, size_t* bytes) {
  if (int rc = check_matrix(w)) return rc;
  FP4_REQUIRE(bytes != nullptr && tokens >= 0, "FP4 product: bad workspace query.");
  *bytes = static_cast<size_t>(plan_linear(*w, tokens).total);
  return PIPER_FP4_OK;
}

int piper_fp4_linear(const piper_fp4_matrix* w, const void* x, int64_t x_stride, int64_t tokens, const int32_t* ends,
                     const float* act_second, int32_t scale_mode, void* y, int32_t dtype, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (int rc = check_matrix(w)) return rc;
  if (int rc = check_buffers(w)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  FP4_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 28) && w->batch <= (int64_t{1} << 20), "FP4 product: too many tokens for one call.");
  if (tokens == 0) return PIPER_FP4_OK;
  FP4_REQUIRE(x != nullptr && y != nullptr, "FP4 product: null input or output.");
  FP4_REQUIRE(x_stride >= w->cols || tokens == 1, "FP4 product: rows of the input overlap.");
  FP4_REQUIRE(ends != nullptr || w->batch == 1, "FP4 product: several matrices need the ends of their rows.");
  FP4_REQUIRE(scale_mode >= 0 && scale_mode <= 3, "Unsupported MX scaling mode id.");
  FP4_REQUIRE(act_second == nullptr || w->format == PIPER_FP4_NV, "MXFP4 activations have no second-level scale.");
  const LinearPlan p = plan_linear(*w, tokens);
  if (p.total > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(p.total) || !aligned(workspace, 256)))
    return fail(PIPER_FP4_EWORKSPACE, "FP4 product: workspace missing, too small or not 256-byte aligned.");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const bool x_vec = aligned(x, 32) && (x_stride * static_cast<int64_t>(width(dtype))) % 32 == 0;

  fp4::LinearArgs a{};
  a.w_scale = static_cast<const uint8_t*>(w->scale);
  a.w_second = w->second;
  a.x_second = act_second;
  a.x = x;
  a.x_stride = x_stride;
  a.groups = {ends, tokens, static_cast<int32_t>(w->batch), static_cast<int32_t>((w->rows + 127) / 128)};
  a.y = y;
  a.rows = static_cast<int32_t>(w->rows);
  a.cols = static_cast<int32_t>(w->cols);
  a.k_steps = static_cast<int32_t>((w->cols + 63) / 64);
  a.scale_tiles = static_cast<int32_t>(p.scale_tiles);
  a.split = p.split;
  a.early = !p.move_codes;
  a.vec = aligned(y, 16) && w->rows % 8 == 0;
  a.x_vec = x_vec;
  a.scale_mode = scale_mode;
  a.scale_cols = static_cast<int32_t>(w->cols / block_of(*w));
  if (w->swizzled) {
    // a K step reads two or four scales of a tile: with whole steps no padding is read
    const bool bulk = w->cols % 64 == 0 && aligned(w->scale, 16);
    a.scale_source = bulk ? fp4::kScalesBulk : fp4::kScalesTiles;
    a.scale_piece = aligned(w->scale, 16) ? 16 : 1;
  } else {
    a.scale_source = fp4::kScalesRows;
    for (a.scale_piece = 16; a.scale_piece > 1 && (a.scale_cols % a.scale_piece != 0 || !aligned(w->scale, a.scale_piece));)
      a.scale_piece /= 2;
  }
  const int64_t items = token_tiles(tokens, ends == nullptr ? 0 : w->batch, p.bn) * a.groups.row_tiles;
  a.items = static_cast<int32_t>(items);
  FP4_REQUIRE(items < (int64_t{1} << 31) / fp4::kMaxSplit, "FP4 product: too many tiles for one call.");

  fp4::QuantArgs q{};
  int64_t token_blocks = 0;
  int lane_rows = 1;
  if (!p.fused) {
    q.x = x;
    q.x_stride = x_stride;
    q.rows = q.rows_padded = tokens;
    q.batch = 1;
    q.cols = static_cast<int32_t>(w->cols);
    q.units = static_cast<int32_t>(p.k_padded / fp4::kUnit);
    q.vec = x_vec;
    q.codes = ws + p.x_codes;
    q.code_pitch = p.k_padded / 2;
    q.scale = ws + p.x_scale;
    q.scale_cols = static_cast<int32_t>(p.scale_tiles);
    q.swizzled = q.words = q.pairs = q.pad_codes = 1;
    q.scale_mode = scale_mode;
    q.second_mode = act_second != nullptr ? PIPER_FP4_SECOND_GIVEN : PIPER_FP4_SECOND_NONE;
    q.second = const_cast<float*>(act_second);
    q.token_tile = p.bn;
    q.ends = ends;
    q.experts = static_cast<int32_t>(w->batch);
    lane_rows = rows_per_lane(q, dtype);
    q.row_blocks = static_cast<int32_t>(fp4::quant_row_blocks(q, lane_rows));
    token_blocks = fp4::quant_blocks(q, lane_rows);
  }
  a.x_scale = q.scale;
  fp4::RepackArgs r{};
  if (p.move_codes) {
    r.codes = static_cast<const uint8_t*>(w->codes);
    r.codes_out = ws + p.w_codes;
    r.row_bytes = w->cols / 2;
    r.pitch = p.w_code_pitch;
    r.aligned = aligned(w->codes, 8);
    r.pieces = w->batch * w->rows * (p.w_code_pitch / 16);
  }
  const int64_t blocks = token_blocks + (r.pieces + fp4::kQuantThreads - 1) / fp4::kQuantThreads;
  FP4_REQUIRE(blocks < (int64_t{1} << 31), "FP4 product: too many values for one call.");
  const void* codes = p.move_codes ? ws + p.w_codes : w->codes;
  if (!code_map(&a.w_map, codes, p.w_code_pitch, p.w_code_pitch, w->batch * w->rows, fp4::kTileRows) ||
      (!p.fused && !code_map(&a.x_map, q.codes, q.code_pitch, q.code_pitch, tokens, p.bn)))
    return fail(PIPER_FP4_ECUDA, "FP4 product: cuTensorMapEncodeTiled failed.");

  cudaError_t e = cudaSuccess;
  if (blocks > 0) {
    auto grid = static_cast<unsigned>(blocks), tokens_grid = static_cast<unsigned>(token_blocks);
#define CALL(D, F)                                                                                            \
  if (lane_rows == 1) fp4::prepare_kernel<D, F, 1><<<grid, fp4::kQuantThreads, 0, s>>>(q, r, tokens_grid);     \
  else fp4::prepare_kernel<D, F, fp4::quant_rows<D>()><<<grid, fp4::kQuantThreads, 0, s>>>(q, r, tokens_grid)
    FP4_DISPATCH(dtype, w->format, CALL);
#undef CALL
    e = launched();
    if (e != cudaSuccess) return cuda_fail("prepare kernel", e);
  }
#define CALL(D, F)                                                    \
  e = p.fused ? launch_linear<D, F, 32, true>(a, items, s)            \
      : p.bn == 32 ? launch_linear<D, F, 32, false>(a, items, s)      \
              : p.bn == 128 ? launch_linear<D, F, 128, false>(a, items, s) : launch_linear<D, F, 192, false>(a, items, s)
  FP4_DISPATCH(dtype, w->format, CALL);
#undef CALL
  return e == cudaSuccess ? PIPER_FP4_OK : cuda_fail("linear kernel", e);
}

int piper_fp4_grad_input_workspace(const piper_fp4_matrix* w, const void* dy, int64_t dy_stride, int64_t tokens,
                                   int32_t dtype, size_t* bytes) {
  if (int rc = check_matrix(w)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  FP4_REQUIRE(bytes != nullptr && tokens >= 0, "FP4 gradient: bad workspace query.");
  *bytes = static_cast<size_t>(plan_grad(*w, dy, dy_stride, tokens, dtype).total);
  return PIPER_FP4_OK;
}

int piper_fp4_grad_input(const piper_fp4_matrix* w, const void* dy, int64_t dy_stride, int64_t tokens,
                         const int32_t* ends, void* dx, int32_t dtype, void* workspace, size_t workspace_bytes,
                         void* stream) {
  if (int rc = check_matrix(w)) return rc;
  if (int rc = check_buffers(w)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  FP4_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 29), "FP4 gradient: too many tokens for one call.");
  if (tokens == 0) return PIPER_FP4_OK;
  FP4_REQUIRE(dy != nullptr && dx != nullptr, "FP4 gradient: null gradient or output.");
  FP4_REQUIRE(dy_stride >= w->rows || tokens == 1, "FP4 gradient: rows of the gradient overlap.");
  FP4_REQUIRE(ends != nullptr || w->batch == 1, "FP4 gradient: several matrices need the ends of their rows.");
  const GradPlan p = plan_grad(*w, dy, dy_stride, tokens, dtype);
  if (p.total > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(p.total) || !aligned(workspace, 256)))
    return fail(PIPER_FP4_EWORKSPACE, "FP4 gradient: workspace missing, too small or not 256-byte aligned.");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);

  fp4::GradArgs a{};
  a.codes = static_cast<const uint8_t*>(w->codes);
  a.scale = static_cast<const uint8_t*>(w->scale);
  a.second = w->second;
  const GradTile tile = grad_tile(*w, tokens, p.terms, ends != nullptr);
  a.groups = {ends, tokens, static_cast<int32_t>(w->batch), static_cast<int32_t>((w->cols + 128 * tile.rows - 1) / (128 * tile.rows))};
  a.dx = dx;
  a.code_pitch = w->cols / 2;
  a.rows = static_cast<int32_t>(w->rows);
  a.cols = static_cast<int32_t>(w->cols);
  a.swizzled = w->swizzled != 0;
  a.scale_cols = scale_cols(*w);
  a.terms = p.terms;
  a.split = tile.split;
  a.vec = aligned(dx, 16) && w->cols % 8 == 0;
  a.piece = aligned(w->codes, 16) && a.code_pitch % 16 == 0 ? 16 : aligned(w->codes, 8) ? 8 : 1;

  const int bn = tile.bn;
  const void* src = p.move ? workspace : dy;
  const int64_t pitch = p.move ? p.pitch : tokens > 1 ? dy_stride : up(w->rows, 8);
  if (!encode_map(&a.dy_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, src, w->rows, p.terms * tokens, pitch * 2, fp4::kGradStageRows, bn))
    return fail(PIPER_FP4_ECUDA, "FP4 gradient: cuTensorMapEncodeTiled failed.");
  const int64_t items = tile.items;
  const int64_t split_blocks = tokens * ((w->rows + 255) / 256);
  FP4_REQUIRE(items < (int64_t{1} << 31) / fp4::kMaxSplit && split_blocks < (int64_t{1} << 31), "FP4 gradient: too many tiles for one call.");
  cudaError_t e = cudaSuccess;
  if (p.move) {
    auto kernel = dtype == PIPER_FP4_BF16 ? fp4::split_kernel<fp4::kBF16> : fp4::split_kernel<fp4::kF32>;
    kernel<<<static_cast<unsigned>(split_blocks), 256, 0, s>>>(dy, dy_stride, tokens, a.rows, p.pitch,
                                                               static_cast<__nv_bfloat16*>(workspace));
    if ((e = launched()) != cudaSuccess) return cuda_fail("split kernel", e);
  }
#define CALL(D, F)                                       \
  e = bn == 64 ? launch_grad<D, F, 64, 1>(a, items, s)   \
               : tile.rows == 1 ? launch_grad<D, F, 256, 1>(a, items, s) : launch_grad<D, F, 256, 2>(a, items, s)
  FP4_DISPATCH(dtype, w->format, CALL);
#undef CALL
  return e == cudaSuccess ? PIPER_FP4_OK : cuda_fail("gradient kernel", e);
}

int piper_fp4_linear_plan(const piper_fp4_matrix* w, int64_t tokens, piper_fp4_plan* plan) {
  if (int rc = check_matrix(w)) return rc;
  FP4_REQUIRE(plan != nullptr && tokens > 0, "FP4 product: bad plan query.");
  const LinearPlan p = plan_linear(*w, tokens);
  *plan = {p.bn, 128, p.split, p.fused};
  return PIPER_FP4_OK;
}

int piper_fp4_grad_input_plan(const piper_fp4_matrix* w, int64_t tokens, int32_t grouped, int32_t dtype, piper_fp4_plan* plan) {
  if (int rc = check_matrix(w)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  FP4_REQUIRE(plan != nullptr && tokens > 0 && (grouped != 0 || w->batch == 1), "FP4 gradient: bad plan query.");
  const GradTile t = grad_tile(*w, tokens, grad_terms(dtype), grouped != 0);
  *plan = {t.bn, 128 * t.rows, t.split, 0};
  return PIPER_FP4_OK;
}

const char* piper_fp4_last_error(void) { return g_error; }

int piper_fp4_device_status(void* stream, uint32_t* status) {
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail("cudaStreamSynchronize", e);
  unsigned int v = 0, zero = 0;
  e = cudaMemcpyFromSymbol(&v, pm::g_status, sizeof(v));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(pm::g_status, &zero, sizeof(zero));
  if (e != cudaSuccess) return cuda_fail("status word", e);
  if (status) *status = v;
  return v == 0 ? PIPER_FP4_OK : fail(PIPER_FP4_ETIMEOUT, "a bounded device-side wait timed out.");
}

const char* piper_fp4_version(void) { return "piper-fp4 0.1 sm_100a"; }

uint64_t piper_fp4_launches(void) { return g_launches.load(std::memory_order_relaxed); }

}  // extern "C"
