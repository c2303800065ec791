/*
 * mm_group_norm.h -- C ABI of the gated group norm of libmm_scan.so (gfx950), channels last, forward and
 * backward: the norm behind a linear-attention or state-space layer.
 *
 *   h = x, or x * silu(z) with MM_GATE_BEFORE
 *   n = (h - mean) / sqrt(var + eps)      mean, var over each group of channels / n_groups channels of a row;
 *                                         with is_rms: h / sqrt(mean(h^2) + eps)
 *   a = n * weight + bias
 *   y = a, a * silu(z) with MM_GATE_AFTER, or silu(a) with MM_GATE_ACT
 *
 * The statistics run over one row (token): a causal model cannot take them over tokens. They are float32,
 * var as the mean square of h - mean. Rows are `channels` contiguous elements. Conventions as in mm_scan.h.
 */
#ifndef MM_GROUP_NORM_H_
#define MM_GROUP_NORM_H_

#include <stdint.h>

#include "mm_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest channels / n_groups. */
#define MM_GROUP_NORM_MAX_GROUP 16384

typedef enum mm_gate {
    MM_GATE_NONE = 0,
    MM_GATE_AFTER = 1,   /* z */
    MM_GATE_BEFORE = 2,  /* z */
    MM_GATE_ACT = 3      /* no z */
} mm_gate;

typedef struct mm_group_norm_params {
    int64_t rows, channels, n_groups;
    mm_dtype itype;              /* x, z, out, dout, dx, dz */
    mm_dtype wtype;              /* weight, bias, dweight, dbias */
    float eps;
    int32_t is_rms;
    mm_gate gate;
    const void *x, *z;           /* (rows, channels); z as the gate needs */
    const void *weight, *bias;   /* (channels,) contiguous, or NULL (1 and 0) */
    void *out;                   /* contiguous (rows, channels) */
    int64_t x_row_stride, z_row_stride;

    /* Backward only. */
    const void *dout;            /* (rows, channels) */
    int64_t dout_row_stride;
    void *dx, *dz;               /* contiguous (rows, channels); dz with z */
    void *dweight, *dbias;       /* (channels,) or NULL */
    void *workspace;             /* mm_group_norm_bwd_workspace_size() bytes, 16-byte aligned */
    int64_t workspace_bytes;
} mm_group_norm_params;

int mm_group_norm_fwd(const mm_group_norm_params *params, void *stream);
/* Workspace bytes (0: none needed). They depend on which pointers are set, on the alignment of the tensors' and on their row
 * strides, and on the current device's compute-unit count: query with the call's own parameters, its device current. */
int64_t mm_group_norm_bwd_workspace_size(const mm_group_norm_params *params);
int mm_group_norm_bwd(const mm_group_norm_params *params, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MM_GROUP_NORM_H_ */
