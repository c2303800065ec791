/*
 * mm_delta.h -- C ABI of the gated delta rule of libmm_scan.so (gfx950).
 *
 *   S'_t = exp(log_decay_t) S_{t-1}                     S: (dk, dv) per batch row and head, float32
 *   z_t  = v_t - S'_t^T k_t
 *   S_t  = S'_t + beta_t k_t z_t^T
 *   o_t  = scale * S_t^T q_t
 *
 * the recurrence of layers that replace what their state holds under a key instead of adding to it. q and k are shared by the
 * nheads / n_groups heads of a group, as the scan's B and C are. The forward and backward run in chunks on the matrix cores;
 * mm_delta_update is the single-token form on a kept state. Keys are meant to have norm 1 and beta to lie in 0 .. 2 (the state's
 * transition I - beta k k^T then does not grow); the kernels take any.
 *
 * log_decay may be NULL (no decay), and is meant to be <= 0. -inf forgets the state (a document's first token); values below
 * -128 count as -128, whose exponential is 0 in float32, values above 128 as 128, whose exponential is infinite. NaN stays NaN.
 *
 * Infinities and NaN: outputs and states of mm_delta_fwd and mm_delta_update are what the recurrence makes of them (chunks that one
 * reaches run token by token, many times slower). In the gradients of its (batch row, head) what one reaches is NaN or infinite, and
 * other elements may be NaN.
 *
 * Conventions as in mm_scan.h: device pointers, element strides, outputs allocated by the caller, nothing is synchronised or
 * allocated, 0 or a code of mm_scan.h is returned and mm_last_error() has the text. The innermost dimension (dk or dv) of q, k, v,
 * dout and of every output is contiguous; states are contiguous (batch, nheads, dk, dv). Sequence strides are 0 to 2^22 - 1
 * elements (nheads * dk and nheads * dv too in the backward), seqlen is at most 2^23, batch * nheads at most 2^20
 * (mm_delta_update: 2^23 - 1); else MM_ERR_UNSUPPORTED.
 */
#ifndef MM_DELTA_H_
#define MM_DELTA_H_

#include <stdint.h>

#include "mm_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest dk and dv. */
#define MM_DELTA_MAX_DIM 128

typedef struct mm_delta_fwd_params {
    int64_t batch, seqlen, n_groups, nheads, dk, dv;
    mm_dtype itype;              /* q, k, v, out */
    mm_dtype gtype, btype;       /* log_decay; beta */
    float scale;
    const void *q, *k;           /* (batch, seqlen, n_groups, dk) */
    const void *v;               /* (batch, seqlen, nheads, dv) */
    const void *beta;            /* (batch, seqlen, nheads); strides may be 0 */
    const void *log_decay;       /* (batch, seqlen, nheads) or NULL (zeros); strides may be 0 */
    const float *initial_state;  /* (batch, nheads, dk, dv) or NULL (zeros) */
    void *out;                   /* (batch, seqlen, nheads, dv) */
    float *last_state;           /* (batch, nheads, dk, dv) or NULL */
    void *segment_states;        /* mm_delta_segment_states_size() bytes, 16-byte aligned, written for the backward; or NULL */
    int64_t segment_states_bytes;
    void *workspace;             /* mm_delta_fwd_workspace_size() bytes, 16-byte aligned (required) */
    int64_t workspace_bytes;
    int64_t q_batch_stride, q_seq_stride, q_group_stride;
    int64_t k_batch_stride, k_seq_stride, k_group_stride;
    int64_t v_batch_stride, v_seq_stride, v_head_stride;
    int64_t b_batch_stride, b_seq_stride, b_head_stride;
    int64_t g_batch_stride, g_seq_stride, g_head_stride;
    int64_t out_batch_stride, out_seq_stride, out_head_stride;
} mm_delta_fwd_params;

typedef struct mm_delta_bwd_params {
    int64_t batch, seqlen, n_groups, nheads, dk, dv;
    mm_dtype itype;              /* q, k, v, dout, dq, dk_out, dv_out */
    mm_dtype gtype, btype;       /* log_decay, dlog_decay; beta, dbeta */
    float scale;
    const void *q, *k, *v, *beta, *log_decay;
    const float *initial_state;  /* as in the forward */
    const void *dout;            /* (batch, seqlen, nheads, dv) */
    const float *dlast_state;    /* (batch, nheads, dk, dv) or NULL (zeros) */
    void *dq, *dk_out;           /* contiguous (batch, seqlen, n_groups, dk) */
    void *dv_out;                /* contiguous (batch, seqlen, nheads, dv) */
    void *dbeta;                 /* contiguous (batch, seqlen, nheads) */
    void *dlog_decay;            /* contiguous (batch, seqlen, nheads), or (nheads,) with decay_per_head; or NULL */
    float *dinitial_state;       /* (batch, nheads, dk, dv) or NULL */
    int32_t decay_per_head;      /* log_decay is one value per head: dlog_decay is summed over batch and seqlen */
    const void *segment_states;  /* what the forward left there, after a call with the same sizes, inputs and device, or NULL
                                  * (computed again) */
    int64_t segment_states_bytes;   /* as in that call */
    void *workspace;             /* mm_delta_bwd_workspace_size() bytes, 16-byte aligned (required) */
    int64_t workspace_bytes;
    int64_t q_batch_stride, q_seq_stride, q_group_stride;
    int64_t k_batch_stride, k_seq_stride, k_group_stride;
    int64_t v_batch_stride, v_seq_stride, v_head_stride;
    int64_t b_batch_stride, b_seq_stride, b_head_stride;
    int64_t g_batch_stride, g_seq_stride, g_head_stride;
    int64_t do_batch_stride, do_seq_stride, do_head_stride;
} mm_delta_bwd_params;

typedef struct mm_delta_update_params {
    int64_t batch, n_groups, nheads, dk, dv;
    mm_dtype itype;              /* q, k, v, out */
    mm_dtype gtype, btype;       /* log_decay; beta */
    float scale;
    float *state;                /* (batch, nheads, dk, dv), read and written; the last dimension contiguous, no two
                                  * elements in one place */
    const void *q, *k;           /* (batch, n_groups, dk) */
    const void *v;               /* (batch, nheads, dv) */
    const void *beta;            /* (batch, nheads); strides may be 0 */
    const void *log_decay;       /* (batch, nheads) or NULL (zeros); strides may be 0 */
    void *out;                   /* contiguous (batch, nheads, dv) */
    int64_t state_batch_stride, state_head_stride, state_dk_stride;
    int64_t q_batch_stride, q_group_stride;
    int64_t k_batch_stride, k_group_stride;
    int64_t v_batch_stride, v_head_stride;
    int64_t b_batch_stride, b_head_stride;
    int64_t g_batch_stride, g_head_stride;
} mm_delta_update_params;

/* Workspace bytes (0: none needed, or sizes that the call refuses). They depend on the sizes and on the current device's
 * compute-unit count: query with the device of the call current. They also depend on whether segment_states and the backward's
 * dlog_decay are NULL: query with those pointers set as in the call. segment_states' own size is 0 where rows are not cut: leave it NULL
 * then. A call refuses segment_states of any other size than the query's, as after a change of MM_DELTA_SEGMENTS (the number of
 * segments, for measurements) between the two. */
int64_t mm_delta_fwd_workspace_size(const mm_delta_fwd_params *params);
int64_t mm_delta_segment_states_size(const mm_delta_fwd_params *params);
int64_t mm_delta_bwd_workspace_size(const mm_delta_bwd_params *params);

int mm_delta_fwd(const mm_delta_fwd_params *params, void *stream);
/* Gradients of q, k, v, beta, log_decay and initial_state for dout and dlast_state. */
int mm_delta_bwd(const mm_delta_bwd_params *params, void *stream);
/* One token: state in place, out. Calls on one state must be ordered. */
int mm_delta_update(const mm_delta_update_params *params, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MM_DELTA_H_ */
