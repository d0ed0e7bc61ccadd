/* piper_routing.h - C ABI of expert routing and of the exchange of tokens (libpiper_routing.so, sm_100a).
 *
 * route: each token's `top_k` experts from a router's logits, their weights,
 * and the order of all choices by expert, which the grouped products of
 * piper_fp4.h and piper_int8.h take. dispatch and combine copy tokens to their
 * places in that order and add the experts' results up again.
 *
 * Every pointer is a device pointer. Calls enqueue on `stream`, allocate
 * nothing and do not synchronise. They return 0 or one of the codes below;
 * piper_routing_last_error() holds the message. Arguments are checked before
 * anything is enqueued.
 */
#ifndef PIPER_ROUTING_H
#define PIPER_ROUTING_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { PIPER_ROUTING_OK = 0, PIPER_ROUTING_EINVAL = 1, PIPER_ROUTING_ECUDA = 2, PIPER_ROUTING_EWORKSPACE = 3 };
enum { PIPER_ROUTING_BF16 = 0, PIPER_ROUTING_F16 = 1, PIPER_ROUTING_F32 = 2 };
enum { PIPER_ROUTING_SOFTMAX = 0, PIPER_ROUTING_SIGMOID = 1 };
enum { PIPER_ROUTING_MAX = 0, PIPER_ROUTING_TOP2 = 1 };
enum { PIPER_ROUTING_MAX_EXPERTS = 1024, PIPER_ROUTING_MAX_TOP_K = 32, PIPER_ROUTING_MAX_GROUPS = 32 };

typedef struct piper_routing_config {
  int64_t tokens;
  int32_t experts, top_k;
  int32_t scoring;            /* PIPER_ROUTING_SOFTMAX or _SIGMOID */
  int32_t groups, top_groups; /* groups of experts / groups neighbours; 1, 1: all of them */
  int32_t group_score;        /* a group's best choice score (PIPER_ROUTING_MAX) or its two best added up (_TOP2) */
  int32_t renormalize;        /* weights of a token add up to `scale` */
  float scale;
} piper_routing_config;

/* Scratch bytes of piper_routing_route (0: none), 16-byte aligned. */
int piper_routing_workspace(const piper_routing_config* c, size_t* bytes);

/* logits (tokens, experts), rows `stride` values apart. `bias`: fp32
 * (experts), added to the scores for the choice alone; or NULL. `mask`: bytes
 * (tokens), zero for a token that gets no expert; or NULL. Results: weights
 * fp32 and experts int32 (tokens, top_k), the best choice first, 0 and -1
 * where there is none; ends int32 (experts); rows int32 (tokens, top_k), the
 * place of each choice in the order by expert, or -1; source int32
 * (tokens * top_k), the choice (token * top_k + slot) at each place, or -1. */
int piper_routing_route(const piper_routing_config* c, const void* logits, int64_t stride, int32_t dtype,
                        const float* bias, const uint8_t* mask, float* weights, int32_t* experts, int32_t* ends,
                        int32_t* rows, int32_t* source, void* workspace, size_t workspace_bytes, void* stream);

/* The logits' gradient (tokens, experts) of type `dtype` from that of the
 * weights (fp32), for the experts that piper_routing_route chose. */
int piper_routing_route_grad(const piper_routing_config* c, const void* logits, int64_t stride, int32_t dtype,
                             const int32_t* experts, const float* grad, void* dlogits, void* stream);

/* How tokens and choices lie: rows (tokens, top_k) as above, `total` the
 * number of places in use (the last of the ends; all of them where it is
 * larger). A row outside [0, total) counts as none. Each place in [0, total)
 * is one row: what two name, or none, is left undefined in out and dy. */
typedef struct piper_routing_exchange {
  int64_t tokens;
  int32_t top_k;
  int32_t hidden; /* values of a token */
  int32_t dtype;
  const int32_t* rows;
  const int32_t* total;
} piper_routing_exchange;

/* out[rows[t, j]] = x[t]: out is (tokens * top_k, hidden), zero from `total` on. */
int piper_routing_dispatch(const piper_routing_exchange* e, const void* x, int64_t x_stride, void* out, void* stream);

/* out[t] = sum over j of weights[t, j] * y[rows[t, j]], in fp32 in the order
 * of j, rounded once; without weights they are 1. */
int piper_routing_combine(const piper_routing_exchange* e, const void* y, int64_t y_stride, const float* weights,
                          void* out, void* stream);

/* dy[rows[t, j]] = weights[t, j] * dout[t], zero from `total` on;
 * dweights[t, j] = sum over h of dout[t, h] * y[rows[t, j], h], in fp32. */
int piper_routing_combine_grad(const piper_routing_exchange* e, const void* y, int64_t y_stride, const float* weights,
                               const void* dout, int64_t dout_stride, void* dy, float* dweights, void* stream);

/* Message of the calling thread's last failed call ("" if none). */
const char* piper_routing_last_error(void);

const char* piper_routing_version(void);

/* Kernels that this process has launched through this library. */
uint64_t piper_routing_launches(void);

#ifdef __cplusplus
}
#endif

#endif /* PIPER_ROUTING_H */
