/* piper_fp4.h - C ABI of the 4-bit floating-point operators (libpiper_fp4.so, sm_100a).
 *
 * Quantisation, products and gradients over the two packed FP4 layouts that
 * the merges of piper_merge.h read and write:
 *
 *   MXFP4  e2m1 codes, 32 of a row share one e8m0 scale (a power of two);
 *   NVFP4  e2m1 codes, 16 of a row share one e4m3 scale, optionally with one
 *          fp32 second-level scale over the whole matrix.
 *
 * Scales are not negative: products take an e4m3 scale's magnitude.
 * Codes are packed two to a byte, the even column in the low nibble. Scales
 * are row-major (rows x cols / block) or swizzled: tiles of 128 rows x 4
 * scales, byte (r % 32) * 16 + (r / 32) * 4 + c, tiles row-major with both
 * sides rounded up. A matrix may be a stack of `batch` equal ones (experts).
 *
 * Every pointer is a device pointer. Calls enqueue on `stream`, allocate
 * nothing and do not synchronise. They return 0 or one of the codes below;
 * piper_fp4_last_error() holds the message. Arguments are checked before
 * anything is enqueued.
 */
#ifndef PIPER_FP4_H
#define PIPER_FP4_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  PIPER_FP4_OK = 0,
  PIPER_FP4_EINVAL = 1,
  PIPER_FP4_ECUDA = 2,
  PIPER_FP4_EWORKSPACE = 3,
  PIPER_FP4_ETIMEOUT = 4
};

enum { PIPER_FP4_MX = 0, PIPER_FP4_NV = 1 };
enum { PIPER_FP4_BF16 = 0, PIPER_FP4_F32 = 2 };
/* How the e8m0 exponent follows a block's maximum (MXFP4). */
enum { PIPER_FP4_FLOOR = 0, PIPER_FP4_RCEIL = 1, PIPER_FP4_CEIL = 2, PIPER_FP4_EVEN = 3 };
/* Second-level scale of a quantisation: none, read from `second`, or computed
 * as max(max|x| / 2688, 2^-23) over the finite values of each matrix of the
 * batch and written there. */
enum { PIPER_FP4_SECOND_NONE = 0, PIPER_FP4_SECOND_GIVEN = 1, PIPER_FP4_SECOND_COMPUTE = 2 };

/* Matrices of at most so many values need no room for maxima (piper_fp4_quantize). */
enum { PIPER_FP4_SMALL_MATRIX = 65536 };

/* A packed matrix, or `batch` of them one after another (experts). */
typedef struct piper_fp4_matrix {
  void* codes;    /* (batch, rows, cols / 2) */
  void* scale;    /* (batch, rows, cols / block), or swizzled */
  float* second;  /* fp32 (batch), or NULL; NVFP4 only */
  int64_t batch, rows, cols;
  int32_t format;   /* PIPER_FP4_MX or PIPER_FP4_NV */
  int32_t swizzled; /* layout of `scale` */
} piper_fp4_matrix;

/* Quantises x (batch * rows rows of `cols` values, `x_stride` values apart)
 * into m's buffers. Swizzle padding is zeroed. `maxima`: scratch of `batch`
 * words when second_mode is PIPER_FP4_SECOND_COMPUTE and a matrix has more
 * than PIPER_FP4_SMALL_MATRIX values; else it is not used. */
int piper_fp4_quantize(const piper_fp4_matrix* m, const void* x, int64_t x_stride, int32_t dtype, int32_t scale_mode,
                       int32_t second_mode, uint32_t* maxima, void* stream);

/* y (batch, rows, cols) = the values that m's codes and scales stand for,
 * formed in fp32 and rounded once. */
int piper_fp4_dequantize(const piper_fp4_matrix* m, void* y, int32_t dtype, void* stream);

/* Scratch bytes that piper_fp4_linear / piper_fp4_grad_input need (0: none). */
int piper_fp4_linear_workspace(const piper_fp4_matrix* w, int64_t tokens, size_t* bytes);
int piper_fp4_grad_input_workspace(const piper_fp4_matrix* w, const void* dy, int64_t dy_stride, int64_t tokens,
                                   int32_t dtype, size_t* bytes);

/* y[t] = w . quantised(x[t]): y is (tokens, rows), x is (tokens, cols) with
 * rows `x_stride` values apart. x is quantised in w's format, with
 * `scale_mode` for MXFP4 and the optional second-level scale `act_second` for
 * NVFP4. With `ends` (int32, w->batch of them, non-decreasing) matrix e
 * multiplies the rows [ends[e-1], ends[e]); rows past the last end become
 * zero. An end below one before it counts as that one, one past the tokens as
 * theirs. Without it w->batch is 1. The workspace is 256-byte aligned. */
int piper_fp4_linear(const piper_fp4_matrix* w, const void* x, int64_t x_stride, int64_t tokens, const int32_t* ends,
                     const float* act_second, int32_t scale_mode, void* y, int32_t dtype, void* workspace,
                     size_t workspace_bytes, void* stream);

/* dx[t] = transposed(w) . dy[t]: dx is (tokens, cols), dy is (tokens, rows)
 * with rows `dy_stride` values apart; `ends` as above. */
int piper_fp4_grad_input(const piper_fp4_matrix* w, const void* dy, int64_t dy_stride, int64_t tokens,
                         const int32_t* ends, void* dx, int32_t dtype, void* workspace, size_t workspace_bytes,
                         void* stream);

/* How the product of `tokens` tokens, or its gradient, runs on the current
 * device: what its tiles are and who works on them. Results do not depend on
 * it but for the order of sums. */
typedef struct piper_fp4_plan {
  int32_t tile_tokens;
  int32_t tile_columns; /* of y, or of dx */
  int32_t split;        /* blocks that share the sums of a tile */
  int32_t fused;        /* the product quantises its tokens itself */
} piper_fp4_plan;

int piper_fp4_linear_plan(const piper_fp4_matrix* w, int64_t tokens, piper_fp4_plan* plan);
/* `grouped`: with the ends of the matrices' rows. */
int piper_fp4_grad_input_plan(const piper_fp4_matrix* w, int64_t tokens, int32_t grouped, int32_t dtype,
                              piper_fp4_plan* plan);

/* Message of the calling thread's last failed call ("" if none). */
const char* piper_fp4_last_error(void);

/* Reads and clears the device-side error word (nonzero when a bounded wait
 * timed out). Synchronises `stream`. */
int piper_fp4_device_status(void* stream, uint32_t* status);

const char* piper_fp4_version(void);

/* Kernels that this process has launched through this library. */
uint64_t piper_fp4_launches(void);

#ifdef __cplusplus
}
#endif

#endif /* PIPER_FP4_H */
