/*
 * mm_layer_norm.h -- C ABI of the residual add with layer norm (or RMS norm) of libmm_scan.so (gfx950), channels last, forward and
 * backward: the norm at a layer's entry.
 *
 *   h = x + residual
 *   n = (h - mean) / sqrt(var + eps)      over a row's channels; with is_rms: h / sqrt(mean(h^2) + eps)
 *   y = n * weight + bias
 *   residual_out = h, rounded to rtype
 *
 * h and the statistics are float32 (var as the mean square of h - mean); the norm is that of h, not of its rounded copy. Rows are
 * `channels` contiguous elements. Conventions as in mm_scan.h.
 */
#ifndef MM_LAYER_NORM_H_
#define MM_LAYER_NORM_H_

#include <stdint.h>

#include "mm_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest row. */
#define MM_LAYER_NORM_MAX_CHANNELS 16384

typedef struct mm_layer_norm_params {
    int64_t rows, channels;
    mm_dtype itype;              /* x, out, dout, dx */
    mm_dtype rtype;              /* residual, residual_out, dresidual_out, dresidual */
    mm_dtype wtype;              /* weight, bias, dweight, dbias */
    float eps;
    int32_t is_rms;
    const void *x;               /* (rows, channels); NULL: residual holds h already (the backward of a kept float32 h) */
    const void *residual;        /* (rows, channels) or NULL (zeros) */
    const void *weight, *bias;   /* (channels,) contiguous, or NULL (1 and 0) */
    void *out;                   /* contiguous (rows, channels) */
    void *residual_out;          /* contiguous (rows, channels) or NULL */
    int64_t x_row_stride, residual_row_stride;

    /* Backward only. */
    const void *dout;            /* (rows, channels) */
    const void *dresidual_out;   /* (rows, channels) or NULL (zeros) */
    int64_t dout_row_stride, dresidual_out_row_stride;
    void *dx;                    /* contiguous (rows, channels) or NULL */
    void *dresidual;             /* contiguous (rows, channels) or NULL */
    void *dweight, *dbias;       /* (channels,) or NULL */
    void *workspace;             /* mm_layer_norm_bwd_workspace_size() bytes, 16-byte aligned */
    int64_t workspace_bytes;
} mm_layer_norm_params;

int mm_layer_norm_fwd(const mm_layer_norm_params *params, void *stream);
/* Workspace bytes (0: none needed). They depend on rows, channels and itype, on whether dweight or dbias is set, and on the current
 * device's compute-unit count: query with the call's own parameters, its device current. */
int64_t mm_layer_norm_bwd_workspace_size(const mm_layer_norm_params *params);
int mm_layer_norm_bwd(const mm_layer_norm_params *params, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MM_LAYER_NORM_H_ */
