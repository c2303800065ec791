// mm_delta_host.h -- arguments and launchers shared by the gated delta rule's translation units.
#pragma once

#include <hip/hip_runtime.h>

#include "mm_delta.h"
#include "mm_linattn_host.h"

namespace mm {
namespace dr {

using la::View;

// One number per token and head (log decays, beta); strides in elements.
struct Gate {
    const void *p;
    mm_dtype type;
    int64_t batch, seq, head;
};

// Tokens of a chunk. (The linear attention's Cfg has the same: 16-bit and float32 tiles of both fit the LDS.)
inline int chunk_tokens(mm_dtype t) { return t == MM_BFLOAT16 ? 64 : 32; }
// 32-wide operands of a chunk's lower triangle of 16 x 16 tiles.
inline int chunk_frags(int tokens) { return tokens == 64 ? 6 : 2; }
// Bytes of a chunk's triangle as operands: three planes of 64 x 16 bytes each.
inline int64_t image_bytes(int tokens) { return int64_t(chunk_frags(tokens)) * 3 * 1024; }
// Of its decays and beta; of its record: images, then those.
constexpr int64_t steps_bytes(int tokens) { return (6 * tokens + 1) * 4 + 12; }
inline int64_t record_bytes(int tokens, int images) { return images * image_bytes(tokens) + steps_bytes(tokens); }

// The argument block of every kernel; each reads what it needs.
struct Args {
    View q, k, v, dout;
    Gate g, beta;                  // g.p NULL: no decay
    int64_t batch, seqlen, heads, chunks;
    int dk, dv, slices;            // slices: workgroups over dv
    float scale;
    char *rec_a, *rec_b;           // [bh][chunk] records (dr_prep): images of P and M, or, for the backward, of P in rec_a and of the
                                   // transposes of both in rec_b
    int rec_a_step;                // bytes of a record of rec_a
    int segs;                      // segments of a row, seg_len tokens each (a multiple of the chunk)
    int64_t seg_len;
    float *maps, *starts;          // [bh][seg][KD][VD + KD], [bh][seg][KD][VD]
    float *back_maps, *back_starts;   // the backward's: [bh][seg][KD][VD] both
    int last_map;                  // the last segment's map too (the backward's)
    int kept_starts;               // maps and starts are there already
    int *flags;                    // [bh]: a row's states are not finite
    const float *s0;               // state before the first token, or NULL
    float *s1;                     // state after the last one, or NULL
    float *states, *z;             // the backward's: [bh][chunk][KD][VD], [bh][chunk * C][VD]
    float *r, *dx;                 // the states' gradients at the chunks' ends, dv before its rounding; sizes as above
    const float *dlast;            // gradient of s1, or NULL
    float *ds0;                    // of s0, or NULL
    float *pbeta;                  // [slice][bh][chunk * C]: a slice's share of dbeta
    void *out;                     // out, or dv
    int out_vec;
    int64_t out_batch, out_seq, out_head;
    void *dq, *dk_out;             // [batch][seqlen][heads][dk], T or float32
    int dqk_f32, dqk_vec;
    void *dbeta, *dg;              // [batch][seqlen][heads]; dg or NULL
    float *dg_sum;                 // [bh][seqlen] instead of dg: one value per head
};

template <typename T> int launch_prep(const Args &a, bool rev, hipStream_t s);
template <typename T> int launch_walk(const Args &a, bool states, hipStream_t s);
template <typename T> int launch_back(const Args &a, hipStream_t s);
template <typename T> int launch_grad(const Args &a, hipStream_t s);

}  // namespace dr
}  // namespace mm
