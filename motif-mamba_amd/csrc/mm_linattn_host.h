// mm_linattn_host.h -- arguments and launchers shared by the linear attention's translation units.
#pragma once

#include <hip/hip_runtime.h>

#include "mm_linattn.h"

namespace mm {
namespace la {

// A (batch, seqlen, heads / share, d) tensor; `vec`: its rows can be read in 16-byte pieces.
struct View {
    const void *p;
    int64_t batch, seq, head;
    int share, vec;
};

struct State {
    float *p;
    int64_t row, col;      // strides
};

// A walk from the front over X, Y (rows of kdim) and V (rows of cdim).
struct WalkArgs {
    View x, y, v, z;       // z: only with the row products (e)
    const void *g;
    mm_dtype gtype;
    int64_t g_batch, g_seq, g_head;
    int64_t batch, seqlen, heads;
    int kdim, cdim, segs;
    int slices;            // the segments' pass: workgroups over V's columns
    int64_t seg_len;       // tokens, a multiple of kBlock
    float scale;
    State s0;              // state the first token (or each segment) starts from, s0_step elements apart
    int64_t s0_step;
    State s1;              // state after the last token
    void *out;             // T, or float32 with out_f32
    int out_f32, out_vec;  // out_vec: 16-byte stores
    int64_t out_batch, out_seq, out_head;
    float *e;              // [bh][seqlen]
    float *ck;             // [bh][blocks][kdim][cdim]: states before token (i + 1) kBlock; the last one after the last token
    int ck_last;
    int64_t blocks;
    float *st, *seg_decay; // the segments' pass: [bh][segs][kdim][cdim], [bh][segs]
};

struct BwdArgs {
    View q, k, v, dout;
    const void *g;
    mm_dtype gtype;
    int64_t g_batch, g_seq, g_head;
    int64_t batch, seqlen, heads;
    int dk, dv, segs;
    int64_t seg_len;
    float scale;
    const float *r0;       // [bh][segs][dk][dv]: the state's gradient at each segment's end; NULL: zeros
    float *dr;             // [bh][dk][dv]: at the first token
    void *dv_out, *dk_out; // [batch][seqlen][heads][dv], [batch][seqlen][heads][dk] (float32 with dk_f32)
    int dk_f32, out_vec;
    float *a, *f;          // [bh][seqlen] each, or NULL: no gradient of the decays
    const float *ck;       // [bh][blocks][dv][dk]
    float *y;              // [bh][blocks][4]
    int has_last;
    int64_t blocks;
};

template <typename T> int launch_walk(const WalkArgs &a, bool dot, hipStream_t s);
template <typename T> int launch_segments(const WalkArgs &a, bool rev, hipStream_t s);
template <typename T> int launch_bwd(const BwdArgs &a, hipStream_t s);
int launch_join(float *st, const float *decay, const float *edge, int segs, int64_t size, int64_t bh, bool rev, hipStream_t s);
int launch_head_sum(const float *part, void *out, mm_dtype t, int64_t rows, int heads, int share, int d, hipStream_t s);
int launch_decay_grad(const BwdArgs &a, const float *e, int C, bool per_head, void *out, mm_dtype gtype, hipStream_t s);
int launch_copy(float *dst, const float *src, int64_t n, hipStream_t s);
int launch_zero_g(void *dst, mm_dtype t, int64_t n, hipStream_t s);

}  // namespace la
}  // namespace mm
