/* piper_int8.h - C ABI of the 8-bit integer products (libpiper_int8.so, sm_100a).
 *
 * Products of tokens with the INT8 weights that the merges of piper_merge.h
 * change, and the products' gradients. A weight is int8 codes with a scale,
 * and optionally a zero point, for each row or for all of it:
 *
 *   value[n, k] = (code[n, k] - zero[n]) * scale[n]      (over_127: scale[n] / 127)
 *
 * A token is quantised by its own largest magnitude a: codes rint(127 x / a),
 * ties to even, scale a / 127. Sums are whole numbers. A token that holds an
 * infinity or a NaN gives a row of NaN. A matrix may be a stack of `batch`
 * equal ones (experts).
 *
 * Every pointer is a device pointer. Calls enqueue on `stream`, allocate
 * nothing and do not synchronise. They return 0 or one of the codes below;
 * piper_int8_last_error() holds the message. Arguments are checked before
 * anything is enqueued.
 */
#ifndef PIPER_INT8_H
#define PIPER_INT8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  PIPER_INT8_OK = 0,
  PIPER_INT8_EINVAL = 1,
  PIPER_INT8_ECUDA = 2,
  PIPER_INT8_EWORKSPACE = 3,
  PIPER_INT8_ETIMEOUT = 4
};

enum { PIPER_INT8_BF16 = 0, PIPER_INT8_F16 = 1, PIPER_INT8_F32 = 2 };

/* Sums of a product fit 32 bits up to so many columns. */
enum { PIPER_INT8_MAX_COLS = 65536 };

/* A weight, or `batch` of them one after another (experts). */
typedef struct piper_int8_matrix {
  const void* codes; /* (batch, rows, cols) int8 */
  const void* scale; /* (batch, rows), or one value */
  const void* zero;  /* int8, as many as scales; or NULL */
  int64_t batch, rows, cols;
  int32_t scale_dtype; /* PIPER_INT8_BF16, _F16 or _F32 */
  int32_t per_row;     /* 0: one scale and zero point, of a single weight */
  int32_t over_127;    /* scales are rows' largest magnitudes: codes / 127 of them */
} piper_int8_matrix;

/* Scratch bytes that piper_int8_linear / piper_int8_grad_input need (0: none).
 * `grouped`: with the ends of the matrices' rows. */
int piper_int8_linear_workspace(const piper_int8_matrix* w, int64_t tokens, int32_t grouped, size_t* bytes);
int piper_int8_grad_input_workspace(const piper_int8_matrix* w, int64_t tokens, int32_t dtype, size_t* bytes);

/* y[t] = w . quantised(x[t]): y is (tokens, rows), x is (tokens, cols) with
 * rows `x_stride` values apart, both of type `dtype`. With `ends` (int32,
 * w->batch of them, non-decreasing) matrix e multiplies the rows
 * [ends[e-1], ends[e]); rows past the last end become zero. An end below one
 * before it counts as that one, one past the tokens as theirs. Without it
 * w->batch is 1. The workspace is 256-byte aligned. */
int piper_int8_linear(const piper_int8_matrix* w, const void* x, int64_t x_stride, int64_t tokens, const int32_t* ends,
                      void* y, int32_t dtype, void* workspace, size_t workspace_bytes, void* stream);

/* dx[t] = transposed(w) . dy[t]: dx is (tokens, cols), dy is (tokens, rows)
 * with rows `dy_stride` values apart; `ends` as above. */
int piper_int8_grad_input(const piper_int8_matrix* w, const void* dy, int64_t dy_stride, int64_t tokens,
                          const int32_t* ends, void* dx, int32_t dtype, void* workspace, size_t workspace_bytes,
                          void* stream);

/* How the product of `tokens` tokens, or its gradient, runs on the current
 * device. Results do not depend on it but for the order of a gradient's sums. */
typedef struct piper_int8_plan {
  int32_t tile_tokens;  /* 8: the product quantises its tokens itself */
  int32_t tile_columns; /* of y, or of dx */
  int32_t split;        /* blocks that share the sums of a tile */
  int32_t blocks;       /* on an SM at a time */
} piper_int8_plan;

int piper_int8_linear_plan(const piper_int8_matrix* w, int64_t tokens, int32_t grouped, piper_int8_plan* plan);
int piper_int8_grad_input_plan(const piper_int8_matrix* w, int64_t tokens, int32_t grouped, int32_t dtype,
                               piper_int8_plan* plan);

/* Message of the calling thread's last failed call ("" if none). */
const char* piper_int8_last_error(void);

/* Reads and clears the device-side error word (nonzero when a bounded wait
 * timed out). Synchronises `stream`. */
int piper_int8_device_status(void* stream, uint32_t* status);

const char* piper_int8_version(void);

/* Kernels that this process has launched through this library. */
uint64_t piper_int8_launches(void);

#ifdef __cplusplus
}
#endif

#endif /* PIPER_INT8_H */
