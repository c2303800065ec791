/*
 * mm_linattn.h -- C ABI of the linear attention with one decay for each head, of libmm_scan.so (gfx950).
 *
 *   S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T          S: (dk, dv) per batch row and head, float32
 *   o_t = scale * S_t^T q_t
 *
 * the recurrence of layers whose state decays by one scalar per head and step (the state-space duals of
 * the selective scan, retention). q and k are shared by the nheads / n_groups heads of a group, as the
 * scan's B and C are. The forward and backward run in chunks on the matrix cores; mm_linattn_update is
 * the single-token form on a kept state.
 *
 * log_decay is meant to be <= 0. -inf forgets the state (a document's first token); values below -128
 * count as -128, whose exponential is 0 in float32, values above 128 as 128, whose exponential is infinite. NaN stays
 * NaN.
 *
 * Infinities: the outputs and states of mm_linattn_fwd and mm_linattn_update, and dq, are what the recurrence makes of them,
 * +-infinity or NaN; in the other gradients what they reach is NaN or infinite. Rows that hold one take some six times as long
 * in mm_linattn_fwd.
 *
 * Conventions as in mm_scan.h: device pointers, element strides, outputs allocated by the caller, nothing
 * is synchronised or allocated, 0 or a code of mm_scan.h is returned and mm_last_error() has the text. The
 * innermost dimension (dk or dv) of q, k, v, dout and of every output is contiguous; states are contiguous
 * (batch, nheads, dk, dv). Sequence strides are 0 to 2^22 - 1 elements (nheads * dk and nheads * dv too in the backward), seqlen is at
 * most 2^23, batch * nheads at most 2^23 - 1 (mm_linattn_update: 2^24 - 1); else MM_ERR_UNSUPPORTED.
 */
#ifndef MM_LINATTN_H_
#define MM_LINATTN_H_

#include <stdint.h>

#include "mm_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest dk and dv. */
#define MM_LINATTN_MAX_DIM 128

typedef struct mm_linattn_fwd_params {
    int64_t batch, seqlen, n_groups, nheads, dk, dv;
    mm_dtype itype;              /* q, k, v, out */
    mm_dtype gtype;              /* log_decay */
    float scale;
    const void *q, *k;           /* (batch, seqlen, n_groups, dk) */
    const void *v;               /* (batch, seqlen, nheads, dv) */
    const void *log_decay;       /* (batch, seqlen, nheads); strides may be 0 */
    const float *initial_state;  /* (batch, nheads, dk, dv) or NULL (zeros) */
    void *out;                   /* (batch, seqlen, nheads, dv) */
    float *last_state;           /* (batch, nheads, dk, dv) or NULL */
    void *workspace;             /* mm_linattn_fwd_workspace_size() bytes, 16-byte aligned. Afterwards it holds the states that
                                  * the row's segments start from. NULL, or fewer bytes: one pass per row, nothing is kept
                                  * (and nothing of it may be handed to the backward as segment_states). */
    int64_t workspace_bytes;
    int64_t q_batch_stride, q_seq_stride, q_group_stride;
    int64_t k_batch_stride, k_seq_stride, k_group_stride;
    int64_t v_batch_stride, v_seq_stride, v_head_stride;
    int64_t g_batch_stride, g_seq_stride, g_head_stride;
    int64_t out_batch_stride, out_seq_stride, out_head_stride;
} mm_linattn_fwd_params;

typedef struct mm_linattn_bwd_params {
    int64_t batch, seqlen, n_groups, nheads, dk, dv;
    mm_dtype itype;              /* q, k, v, dout, dq, dk_out, dv_out */
    mm_dtype gtype;              /* log_decay, dlog_decay */
    float scale;
    const void *q, *k, *v, *log_decay;
    const float *initial_state;  /* as in the forward */
    const void *dout;            /* (batch, seqlen, nheads, dv) */
    const float *dlast_state;    /* (batch, nheads, dk, dv) or NULL (zeros) */
    void *dq, *dk_out;           /* contiguous (batch, seqlen, n_groups, dk) */
    void *dv_out;                /* contiguous (batch, seqlen, nheads, dv) */
    void *dlog_decay;            /* contiguous (batch, seqlen, nheads), or (nheads,) with decay_per_head; or NULL */
    float *dinitial_state;       /* (batch, nheads, dk, dv) or NULL */
    const void *segment_states;  /* the forward's workspace, of the full size, after a call with the same sizes, inputs and
                                  * device, or NULL (computed again) */
    int32_t decay_per_head;      /* log_decay is one value per head: dlog_decay is summed over batch and seqlen */
    void *workspace;             /* mm_linattn_bwd_workspace_size() bytes, 16-byte aligned (required) */
    int64_t workspace_bytes;
    int64_t q_batch_stride, q_seq_stride, q_group_stride;
    int64_t k_batch_stride, k_seq_stride, k_group_stride;
    int64_t v_batch_stride, v_seq_stride, v_head_stride;
    int64_t g_batch_stride, g_seq_stride, g_head_stride;
    int64_t do_batch_stride, do_seq_stride, do_head_stride;
} mm_linattn_bwd_params;

typedef struct mm_linattn_update_params {
    int64_t batch, n_groups, nheads, dk, dv;
    mm_dtype itype;              /* q, k, v, out */
    mm_dtype gtype;              /* log_decay */
    float scale;
    float *state;                /* (batch, nheads, dk, dv), read and written; the last dimension contiguous, no two
                                  * elements in one place */
    const void *q, *k;           /* (batch, n_groups, dk) */
    const void *v;               /* (batch, nheads, dv) */
    const void *log_decay;       /* (batch, nheads); strides may be 0 */
    void *out;                   /* contiguous (batch, nheads, dv) */
    int64_t state_batch_stride, state_head_stride, state_dk_stride;
    int64_t q_batch_stride, q_group_stride;
    int64_t k_batch_stride, k_group_stride;
    int64_t v_batch_stride, v_head_stride;
    int64_t g_batch_stride, g_head_stride;
} mm_linattn_update_params;

/* Workspace bytes (0: none needed). They depend on the sizes and on the current device's compute-unit count: query with
 * the device of the call current. The backward's also depend on whether dlog_decay and segment_states are NULL: query with
 * those pointers set as in the call. */
int64_t mm_linattn_fwd_workspace_size(const mm_linattn_fwd_params *params);
int64_t mm_linattn_bwd_workspace_size(const mm_linattn_bwd_params *params);

int mm_linattn_fwd(const mm_linattn_fwd_params *params, void *stream);
/* Gradients of q, k, v, log_decay and initial_state for dout and dlast_state. */
int mm_linattn_bwd(const mm_linattn_bwd_params *params, void *stream);
/* One token: state in place, out. Calls on one state must be ordered. */
int mm_linattn_update(const mm_linattn_update_params *params, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MM_LINATTN_H_ */
