/*
 * dcc_delta.h -- C-ABI of the gated delta rule (the memory layer of the recurrent policies) in libdcc_hip.so.
 *
 * The reference's recurrent core is a GRU (uav_dcc_control/algos/algo_utils/rnn.py:7-82); this layer stands beside it: every head
 * keeps a matrix S [dk, dv] that is written and corrected by keys and read by queries.  Per row b, head h and token t
 *
 *     S' = m_t exp(g_t) S          m_t = 0 (masks[t,b] == 0): the state restarts from zero, whatever it held (NaN included)
 *     r  = v_t - S'^T k_t          u = beta_t r          S = S' + k_t u^T          o_t = scale * S^T q_t
 *
 *   dcc_delta_fwd     T tokens: o and the last state; optionally the states the gradient starts from (`ckpt`)
 *   dcc_delta_bwd     its gradient for q, k, v, g, beta and the first state
 *   dcc_delta_step    one token (rollout, serving): the state is read and written once, in place if state1 == state0
 *                     (o and state1 lie apart from the operands and from each other)
 *
 * Layout: time-major.  q, k: [T, B, HK, DK], v, o: [T, B, H, DV] in `dtype` (float32, bfloat16 or float16), H a multiple of HK: value
 * head h reads key head h / (H / HK).  g (log decay, <= 0 in use), beta: [T, B, H] float32; masks: [T, B] float32 or NULL (no restarts).
 * The last axis of q, k, v, do is contiguous, the others have strides in ELEMENTS (st_*: t, b, h); so have g, beta (t, b, h) and
 * masks (t, b).  States are contiguous [B, H, DK, DV] float32 and stay in 32 bits.  1 <= DK, DV <= DCC_DELTA_MAX_DIM.
 * exp(g_t) that is 0 in float32 restarts the state like a mask.  Values that are not finite reach what the recurrence, taken token by token,
 * lets them reach: the results of their token and of later ones up to the next restart, the gradients of earlier ones down to the last
 * restart (a chunk of 16 tokens that holds such values takes many times as long).  Finite ones whose sums leave float32's range may reach
 * their whole chunk (chunks start at t = 0, 16, ...).
 *
 * Results lie apart from the operands and from each other (but for a step's state in place).
 *
 * All pointers are device pointers; calls are asynchronous on `stream` and keep nothing; return 0 or a negative DCC_E* code with
 * the message in dcc_last_error().  T == 0 or B == 0 launch nothing except the copy of the state.  Results do not depend on
 * scheduling: no atomics.
 */
#ifndef DCC_DELTA_H
#define DCC_DELTA_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef DCC_API
#if defined(__GNUC__)
#define DCC_API __attribute__((visibility("default")))
#else
#define DCC_API
#endif
#endif

#define DCC_DELTA_MAX_DIM 128
#define DCC_DELTA_F32 0
#define DCC_DELTA_BF16 1
#define DCC_DELTA_F16 2

typedef struct {
    int64_t T, B;                /* tokens, rows */
    int32_t HK, H, DK, DV;       /* key heads, value heads, head sizes */
    int32_t dtype;               /* DCC_DELTA_F32 / BF16 / F16: q, k, v, o and their gradients */
    float scale;                 /* of the output, usually DK^-1/2 */
    const void *q, *k, *v;
    const float *g, *beta;
    const float *masks;          /* NULL: no restarts */
    const float *state0;         /* NULL: zero */
    int64_t st_q[3], st_k[3], st_v[3], st_g[3], st_beta[3], st_masks[2];
    void *o;                     /* contiguous [T, B, H, DV] */
    float *state1;               /* the last state; may be NULL in dcc_delta_fwd */
    float *ckpt;                 /* dcc_delta_fwd: NULL, or dcc_delta_ckpt_floats() floats that dcc_delta_bwd reads */
} dcc_delta_seq;

typedef struct {
    const void *dout;            /* gradient of o, in dtype */
    int64_t st_do[3];
    const float *dstate1;        /* gradient of the last state, contiguous; NULL: zero */
    const float *ckpt;           /* what dcc_delta_fwd left */
    void *dq, *dk, *dv;          /* contiguous [T, B, HK, DK], [T, B, HK, DK], [T, B, H, DV], in dtype */
    float *dg, *dbeta;           /* contiguous [T, B, H] */
    float *dstate0;              /* contiguous, or NULL */
} dcc_delta_grad;

/* Floats of `ckpt` for these sizes (the state at the start of every chunk of 16 tokens); 0 for sizes that are refused. */
DCC_API int64_t dcc_delta_ckpt_floats(const dcc_delta_seq* s);
/* Floats of `workspace` of dcc_delta_fwd / dcc_delta_bwd (0: none needed; NULL is then allowed). */
DCC_API int64_t dcc_delta_fwd_workspace_floats(const dcc_delta_seq* s);
DCC_API int64_t dcc_delta_bwd_workspace_floats(const dcc_delta_seq* s);

DCC_API int dcc_delta_fwd(const dcc_delta_seq* s, float* workspace, void* stream);
DCC_API int dcc_delta_bwd(const dcc_delta_seq* s, const dcc_delta_grad* d, float* workspace, void* stream);
/* One token: s->T == 1; the token strides are not read.  state0 and state1 must be given; equal pointers update in place. */
DCC_API int dcc_delta_step(const dcc_delta_seq* s, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DCC_DELTA_H */
