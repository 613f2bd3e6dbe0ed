/* SunnyNet HIP backend: operators of recurrent language models on device memory.
 *
 * No counterpart in the reference. Like snhip.h this header is not part of the
 * stable ABI. Every call takes DEVICE pointers (the arrays it names below) and a
 * hipStream_t as void* (NULL = the null stream) of the current device, enqueues
 * its work there and returns: no host synchronization, no allocation (workspaces
 * are the caller's), nothing kept between calls, so calls on different streams and
 * captured graphs are independent as long as their arrays are. Status codes are
 * those of snhip_abi.h: SNHIP_E_INVAL for arguments outside the documented ranges,
 * SNHIP_E_DEVICE for a HIP failure.
 */
#ifndef SNHIP_OPS_H
#define SNHIP_OPS_H

#include <stdint.h>

#include "snhip_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define SNHIP_F32   0
#define SNHIP_BF16  1
#define SNHIP_F16   2

/* ------------------------------------------------------ gated delta rule
 * Per sequence and value head h, with a = exp(g):
 *   u_t = beta_t (v_t - a_t S_{t-1}^T k_t)
 *   S_t = a_t S_{t-1} + k_t u_t^T          (K, V)
 *   out_t = scale S_t^T q_t
 * Value head h reads query and key head h / (H / Hk). Sums and states are fp32.
 *
 * Layout: q, k (B,T,Hk,K), v (B,T,H,V) of one element type, the last axis
 * contiguous, the others by the strides below (in elements); g, beta (B,T,H) fp32
 * contiguous; s0, send (N,H,K,V) fp32 contiguous; out (B,T,H,V) contiguous, of the
 * inputs' type. Without cu, N = B sequences of T tokens. With cu (N + 1 int32 on
 * the device, not decreasing, within [0, T]) B is 1 and sequence n holds tokens
 * [cu[n], cu[n+1]); tokens of no sequence are left as they are in every output.
 * Values outside [0, T] are clamped. Two sequences never share a token: cu that
 * decreases is refused by nothing and gives unspecified results (in bounds).
 *
 * Ranges: 1 <= K <= 128, 1 <= V <= 4096, H a multiple of Hk, H <= 65535, N <= 65535,
 * B T < 2^30, H K, H V and every token stride below 2^24 (strides not negative); with
 * workspaces fewer than 2^23 chunks of 32 tokens (B ceil(T / 32), with cu T / 32 + N).
 * g <= 0 is meant (a decay); -inf forgets the state exactly, other values are clamped
 * at -200, where exp(g) is 0 in fp32. Non-finite values reach the results of their
 * sequence and head (in gradients of q and k: of the heads that share theirs) only, as
 * NaN, from the chunk of 32 tokens that holds them on. */
typedef struct SnHipDelta {
    const void* q;
    const void* k;
    const void* v;
    const float* g;
    const float* beta;
    const float* s0;            /* NULL: zeros                                    */
    const int32_t* cu;          /* NULL: B sequences of T tokens                  */
    int64_t q_stride[3];        /* batch, token, head                             */
    int64_t k_stride[3];
    int64_t v_stride[3];
    int64_t B, T, N, Hk, H, K, V;
    int64_t dtype;              /* SNHIP_F32 / BF16 / F16                         */
    double scale;
    float* chunks;              /* workspace: snhip_op_delta_chunk_floats floats  */
    float* states;              /* snhip_op_delta_state_floats floats, written by
                                   the forward for the backward; NULL: not kept.
                                   Both workspaces 16-byte aligned                */
} SnHipDelta;

/* Floats of the two workspaces of a call (the other fields of d are not read); 0 for
 * sizes outside the ranges. */
int64_t snhip_op_delta_chunk_floats(const SnHipDelta* d);
int64_t snhip_op_delta_state_floats(const SnHipDelta* d);

/* out and send (NULL: not wanted). T >= 1, N >= 1. Calls of at most
 * 12 tokens without cu and without states need no workspace (chunks NULL). */
snhip_status snhip_op_delta_fwd_dev(const SnHipDelta* d, void* out, float* send, void* stream);

/* One or a few tokens: the same recurrence token by token, at any T and without
 * workspaces. send must be given; it may be s0 (updated in place), but not overlap it
 * otherwise. */
snhip_status snhip_op_delta_step_dev(const SnHipDelta* d, void* out, float* send, void* stream);

/* Gradients: d as in the forward call, with the chunks and states that it wrote.
 * dout (B,T,H,V) contiguous, of the inputs' type; dsend (N,H,K,V) or NULL (zeros).
 * dq, dk (B,T,Hk,K), dv (B,T,H,V) contiguous, of the inputs' type, dq and dk summed
 * over the value heads that share them; dg, dbeta (B,T,H) fp32; ds0 (N,H,K,V) fp32
 * or NULL. ws: snhip_op_delta_bwd_floats floats (0 outside the ranges), 16-byte aligned. Sums run in a fixed
 * order. */
typedef struct SnHipDeltaGrad {
    const void* dout;
    const float* dsend;
    void* dq;
    void* dk;
    void* dv;
    float* dg;
    float* dbeta;
    float* ds0;
    float* ws;
} SnHipDeltaGrad;
int64_t snhip_op_delta_bwd_floats(const SnHipDelta* d);
snhip_status snhip_op_delta_bwd_dev(const SnHipDelta* d, const SnHipDeltaGrad* gr, void* stream);

/* ------------------------------------------------------------ layer norm
 * y = (x - mean) rstd w + b per row of D values, rstd = 1 / sqrt(var + eps), var
 * over D. x, y (R, D) contiguous of one element type; w, b (D) fp32 or NULL (ones,
 * zeros); mean, rstd (R) fp32 or both NULL (not kept). Statistics in fp32, the
 * variance from the centred values. 1 <= D <= 16384, 1 <= R < 2^31. */
snhip_status snhip_op_norm_fwd_dev(const void* x, const float* w, const float* b, void* y, float* mean,
                                   float* rstd, int64_t R, int64_t D, float eps, int32_t dtype,
                                   void* stream);
/* dx (R, D) of x's type or NULL; dw, db (D) fp32 or NULL each. ws:
 * snhip_op_norm_bwd_floats floats. The sums over rows run in a fixed order. */
int64_t snhip_op_norm_bwd_floats(int64_t R, int64_t D);
snhip_status snhip_op_norm_bwd_dev(const void* dy, const void* x, const float* w, const float* mean,
                                   const float* rstd, void* dx, float* dw, float* db, float* ws, int64_t R,
                                   int64_t D, int32_t dtype, void* stream);

/* -------------------------------------------------------------- sampling
 * The next token of every row of logits (B, V), rows `stride` elements apart, from
 * one random number u in [0, 1) per row. Row settings come from the arrays (B), or,
 * where an array is NULL, from the value beside it:
 *   temperature <= 0: the first maximal logit (a NaN counts as maximal);
 *   else z = logit / temperature in 64 bits, and of the weights exp(z - max z)
 *   top_k in [1, V): those of the k largest z are kept (all that equal the k-th);
 *   top_p in (0, 1): of these, in descending order (equal ones by index), those
 *     before which the kept share is at most top_p;
 *   min_p > 0: those of at least min_p (the largest weight is 1);
 *   the token is the first one up to which the remaining weights sum to more than u
 *   of their total.
 * A row whose weights have no finite positive sum (an infinite or NaN maximum) gives
 * its first maximal logit. Weights are summed as whole numbers of 2^-b of the largest,
 * b = min(51, 62 - ceil(log2 V)) (42 at V = 2^20, 47 at 32000), so a token does not depend
 * on an order of summation, and differs from that of exact weights only where u or a
 * nucleus' end is within V 2^-b of a border, as a share. tokens (B) int32.
 * 1 <= V <= 2^20, B < 2^31. */
typedef struct SnHipSample {
    const void* logits;
    const double* u;
    const double* temperature;
    const int32_t* top_k;
    const double* top_p;
    const double* min_p;
    double temperature0;
    double top_p0;
    double min_p0;
    int64_t top_k0;
    int64_t B, V, stride;
    int64_t dtype;
} SnHipSample;
snhip_status snhip_op_sample_dev(const SnHipSample* s, int32_t* tokens, void* stream);
/* The same, and in drew (B, NULL: not wanted) 1 where u chose the token, 0 where the row
 * gave its first maximal logit. */
snhip_status snhip_op_sample_drew_dev(const SnHipSample* s, int32_t* tokens, int32_t* drew, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SNHIP_OPS_H */
