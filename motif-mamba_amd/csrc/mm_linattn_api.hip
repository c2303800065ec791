// mm_linattn_api.hip -- the linear attention's C entries: argument checks, the plan of a call (segments,
// workspace), and the single-token kernel.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <initializer_list>

#include "mm_common.h"
#include "mm_internal.h"
#include "mm_linattn.h"
#include "mm_linattn_host.h"

namespace mm {
namespace la {

// ---- one token -----------------------------------------------------------------------------------

// S = exp(g) S + k v^T, o = scale S^T q. Bound by the state, read once and written once. A workgroup holds `per`
// rows (dk) of one (batch row, head) at a time: LPR lanes cover a row's dv in 16-byte pieces, so that 64 lanes
// read 1,024 contiguous bytes; each lane's share of o stays in registers and the rows' shares meet in LDS.
// R rows of every lane are loaded before the first is used. 256 x 80 heads of 128 x 64: 262 us, 1.35 GB at 5.1 TB/s (a large
// copy reaches 4.9 here); one sequence: 6 us, the call.
template <typename T, int LPR, int NT>
__global__ void __launch_bounds__(NT) la_update(const mm_linattn_update_params p) {
    constexpr int ROWS = NT / LPR, R = 4;
    __shared__ float4 part[NT / 64][LPR < 64 ? LPR : 64];
    const int64_t bh = blockIdx.x, b = bh / p.nheads, h = bh % p.nheads, grp = h / (p.nheads / p.n_groups);
    const int tid = threadIdx.x, x = 4 * (tid % LPR), row0 = tid / LPR;
    const int dk = int(p.dk), dv = int(p.dv);
    float *s = p.state + b * p.state_batch_stride + h * p.state_head_stride + x;
    const T *q = reinterpret_cast<const T *>(p.q) + b * p.q_batch_stride + grp * p.q_group_stride;
    const T *k = reinterpret_cast<const T *>(p.k) + b * p.k_batch_stride + grp * p.k_group_stride;
    const T *v = reinterpret_cast<const T *>(p.v) + b * p.v_batch_stride + h * p.v_head_stride + x;
    const int n = dv - x < 4 ? dv - x : 4;    // elements of this lane's piece
    const bool vec = n == 4 && (reinterpret_cast<uintptr_t>(p.state) | p.state_dk_stride * 4 | p.state_head_stride * 4 | p.state_batch_stride * 4) % 16 == 0;
    float vv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) vv[e] = e < n ? to_f32(v[e]) : 0.f;
    float g;
    {
        const int64_t at = b * p.g_batch_stride + h * p.g_head_stride;
        switch (p.gtype) {
            case MM_FLOAT32: g = reinterpret_cast<const float *>(p.log_decay)[at]; break;
            case MM_FLOAT16: g = to_f32(reinterpret_cast<const f16_t *>(p.log_decay)[at]); break;
            default: g = to_f32(reinterpret_cast<const bf16_t *>(p.log_decay)[at]);
        }
        g = expf(g < -128.f ? -128.f : g);
    }
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r0 = row0; r0 < dk; r0 += R * ROWS) {
        float w[R][4], kk[R], qq[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = r0 + r * ROWS;
            kk[r] = qq[r] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[r][e] = 0.f;
            if (row < dk) {
                kk[r] = to_f32(k[row]);
                qq[r] = to_f32(q[row]);
                const float *src = s + row * p.state_dk_stride;
                if (vec) {
                    const float4 y = *reinterpret_cast<const float4 *>(src);
                    w[r][0] = y.x; w[r][1] = y.y; w[r][2] = y.z; w[r][3] = y.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < n) w[r][e] = src[e];
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = r0 + r * ROWS;
            if (row >= dk) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[r][e] = __builtin_fmaf(g, w[r][e], kk[r] * vv[e]);
                o[e] = __builtin_fmaf(qq[r], w[r][e], o[e]);
            }
            float *dst = s + row * p.state_dk_stride;
            if (vec) {
                *reinterpret_cast<float4 *>(dst) = make_float4(w[r][0], w[r][1], w[r][2], w[r][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < n) dst[e] = w[r][e];
            }
        }
    }
    // Over the rows a wave holds, then over the waves.
#pragma unroll
    for (int d = LPR; d < 64; d *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], d);
    if (tid % 64 < LPR) part[tid / 64][tid % LPR] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if (tid < LPR && n > 0) {
        float4 y = part[0][tid];
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) {
            const float4 z = part[w][tid];
            y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
        const float r[4] = {y.x * p.scale, y.y * p.scale, y.z * p.scale, y.w * p.scale};
        T *out = reinterpret_cast<T *>(p.out) + bh * dv + x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) out[e] = from_f32<T>(r[e]);
    }
}

template <typename T>
static int launch_update(const mm_linattn_update_params &p, hipStream_t s) {
    const dim3 grid(unsigned(p.batch * p.nheads));
    if (p.dv <= 32) hipLaunchKernelGGL((la_update<T, 8, 256>), grid, dim3(256), 0, s, p);
    else if (p.dv <= 64) hipLaunchKernelGGL((la_update<T, 16, 256>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((la_update<T, 32, 256>), grid, dim3(256), 0, s, p);
    return launch_status("la_update");
}

// ---- the plan of a call --------------------------------------------------------------------------

static size_t size_of(mm_dtype t) { return t == MM_FLOAT32 ? 4 : 2; }
static bool known(mm_dtype t) { return t == MM_FLOAT32 || t == MM_FLOAT16 || t == MM_BFLOAT16; }
static int chunk_of(mm_dtype t) { return t == MM_BFLOAT16 ? 64 : 32; }

constexpr int kBlockTokens = 256;

// A launch takes less than 2^32 threads; a pair has a workgroup of up to 512 (the backward), for one token 256.
constexpr int64_t kMostPairs = (int64_t(1) << 23) - 1, kMostTokenPairs = (int64_t(1) << 24) - 1;

// Segments of a row, by the time that a call takes with n of them, in steps of a chunk of one workgroup alone on its CU
// (about 3.7 us at dk 128, dv 64, bfloat16). Two workgroups on a CU take 1.45 steps per chunk of both. With n > 1 a pass over
// k and v before (0.9 of a step per chunk for few workgroups, 0.5 of one per chunk and CU for many), its join (about 2 steps),
// and the states' traffic, 16 bytes per element and segment at some 4.5 TB/s. Fitted, before the state had its third plane, to: 320 pairs
// (4 x 80 heads), L 4,096: one segment 322 us, two 274 + 128; 192 pairs, L 2,048: one 103 us, three 86 + 45; 64 pairs (dk = dv = 128),
// L 4,096: 100 + 70 us with eight, 240 with one. The same rule serves the other types and sizes, for which nothing was fitted: at
// dk and dv up to 64 a CU holds three workgroups, and float16 and float32 have twice the chunks per token (both sides'
// counts in steps grow alike; the states' traffic then weighs too much). 64 segments at most: the join reads a row's segments one after
// another (64 of 65,536 tokens of 40 heads: 43 us of 1,043, in float32).
static void segments(int64_t pairs, int64_t seqlen, int64_t size, int *segs, int64_t *len) {
    const int64_t cus = device_simds() / 4, blocks = std::max<int64_t>(1, (seqlen + kBlockTokens - 1) / kBlockTokens);
    double best = 0.0;
    for (int64_t n = 1; n <= std::min<int64_t>(blocks, 64); ++n) {
        const int64_t per = (blocks + n - 1) / n, w = (blocks + per - 1) / per;   // blocks per segment, segments
        if (w != n) continue;
        const double steps = double(per) * 4.0;
        const int64_t r = (pairs * n + cus - 1) / cus;
        double t = steps * (1.45 * double(r / 2) + double(r % 2));
        if (n > 1)
            t += steps * std::max(0.9, 0.5 * double(pairs * (n - 1)) / double(cus)) + 2.0 + double(n * pairs * size) * 16.0 / 4.5e12 / 3.7e-6;
        if (n == 1 || t < best) {
            best = t;
            *segs = int(n);
            *len = per * kBlockTokens;
        }
    }
}

static int64_t pad16(int64_t n) { return (n + 15) / 16 * 16; }

static View view(const void *p, mm_dtype t, int64_t b, int64_t s, int64_t h, int share, int64_t d) {
    const int64_t e = int64_t(size_of(t));
    const bool vec = (reinterpret_cast<uintptr_t>(p) | b * e | s * e | h * e | d * e) % 16 == 0;
    return View{p, b, s, h, share, vec ? 1 : 0};
}

static int check(int64_t batch, int64_t seqlen, int64_t groups, int64_t heads, int64_t dk, int64_t dv, mm_dtype it,
                 mm_dtype gt, int64_t pairs) {
    if (!known(it) || !known(gt)) return set_error(MM_ERR_INVALID_ARGUMENT, "linear attention: unknown dtype");
    if (batch < 0 || seqlen < 0 || heads < 0 || dk < 0 || dv < 0) return set_error(MM_ERR_INVALID_ARGUMENT, "linear attention: negative size");
    if (groups < 1 || heads % groups) return set_error(MM_ERR_INVALID_ARGUMENT, "linear attention: nheads must be a multiple of n_groups");
    if (dk < 1 || dv < 1) return set_error(MM_ERR_INVALID_ARGUMENT, "linear attention: dk and dv must be at least 1");
    if (dk > MM_LINATTN_MAX_DIM || dv > MM_LINATTN_MAX_DIM) return set_error(MM_ERR_UNSUPPORTED, "linear attention: dk and dv must be <= 128");
    if (batch > pairs || heads > pairs || batch * heads > pairs) return set_error(MM_ERR_UNSUPPORTED, "linear attention: batch * nheads is too large (at most 2^23 - 1, for one token 2^24 - 1)");
    if (seqlen > (int64_t(1) << 23)) return set_error(MM_ERR_UNSUPPORTED, "linear attention: seqlen must be <= 2^23");
    return MM_OK;
}

// A tile's 64 rows are addressed with 32-bit offsets.
static bool near(std::initializer_list<int64_t> strides) {
    for (const int64_t s : strides)
        if (s < 0 || s >= (int64_t(1) << 22)) return false;
    return true;
}

// No two elements of a state lie in one place: workgroups write them in any order. Each dimension has to step over all that the
// smaller ones span, as views of a contiguous tensor by slices and transposes do.
static bool apart(const mm_linattn_update_params &p) {
    int64_t size[4] = {p.batch, p.nheads, p.dk, p.dv}, step[4] = {p.state_batch_stride, p.state_head_stride, p.state_dk_stride, 1};
    int order[4] = {0, 1, 2, 3};
    for (int64_t &s : step) s = s < 0 ? -s : s;
    std::sort(order, order + 4, [&](int a, int b) { return step[a] < step[b]; });
    int64_t span = 0;
    for (const int d : order) {
        if (size[d] <= 1) continue;
        if (step[d] <= span) return false;
        span += (size[d] - 1) * step[d];
    }
    return true;
}

static int64_t fwd_bytes(const mm_linattn_fwd_params &p, int segs) {
    return segs > 1 ? pad16(p.batch * p.nheads * segs * p.dk * p.dv * 4) + pad16(p.batch * p.nheads * segs * 4) : 0;
}

template <typename T>
static int run_fwd(const mm_linattn_fwd_params &p, hipStream_t s) {
    WalkArgs a = {};
    const int share = int(p.nheads / p.n_groups);
    a.x = view(p.q, p.itype, p.q_batch_stride, p.q_seq_stride, p.q_group_stride, share, p.dk);
    a.y = view(p.k, p.itype, p.k_batch_stride, p.k_seq_stride, p.k_group_stride, share, p.dk);
    a.v = view(p.v, p.itype, p.v_batch_stride, p.v_seq_stride, p.v_head_stride, 1, p.dv);
    a.z = a.v;
    a.g = p.log_decay;
    a.gtype = p.gtype;
    a.g_batch = p.g_batch_stride; a.g_seq = p.g_seq_stride; a.g_head = p.g_head_stride;
    a.batch = p.batch; a.seqlen = p.seqlen; a.heads = p.nheads;
    a.kdim = int(p.dk); a.cdim = int(p.dv);
    segments(p.batch * p.nheads, p.seqlen, p.dk * p.dv, &a.segs, &a.seg_len);
    if (a.segs > 1 && (!p.workspace || p.workspace_bytes < fwd_bytes(p, a.segs))) {
        a.segs = 1;
        a.seg_len = (p.seqlen + kBlockTokens - 1) / kBlockTokens * kBlockTokens;
    }
    const int64_t size = p.dk * p.dv, bh = p.batch * p.nheads;
    if (a.segs > 1) {
        a.st = static_cast<float *>(p.workspace);
        a.seg_decay = reinterpret_cast<float *>(static_cast<char *>(p.workspace) + pad16(bh * a.segs * size * 4));
        a.scale = 1.f;
        if (const int rc = launch_segments<T>(a, false, s)) return rc;
        if (const int rc = launch_join(a.st, a.seg_decay, p.initial_state, a.segs, size, bh, false, s)) return rc;
        a.s0 = State{a.st, p.dv, 1};
    } else {
        a.s0 = State{const_cast<float *>(p.initial_state), p.dv, 1};
    }
    a.s0_step = size;
    a.s1 = State{p.last_state, p.dv, 1};
    a.scale = p.scale;
    a.out = p.out;
    a.out_vec = view(p.out, p.itype, p.out_batch_stride, p.out_seq_stride, p.out_head_stride, 1, p.dv).vec;
    a.out_batch = p.out_batch_stride; a.out_seq = p.out_seq_stride; a.out_head = p.out_head_stride;
    return launch_walk<T>(a, false, s);
}

// The backward's workspace, in order.
struct BwdPlan {
    int segs;
    int64_t seg_len, blocks;
    int64_t st, rt, decay, part, e, a, f, ck, y, bytes;   // byte offsets
};

static BwdPlan plan_bwd(const mm_linattn_bwd_params &p) {
    BwdPlan w = {};
    segments(p.batch * p.nheads, p.seqlen, p.dk * p.dv, &w.segs, &w.seg_len);
    w.blocks = (p.seqlen + kBlockTokens - 1) / kBlockTokens;
    const int64_t bh = p.batch * p.nheads, size = p.dk * p.dv, tok = bh * p.seqlen;
    int64_t at = 0;
    auto take = [&](int64_t floats) {
        const int64_t o = at;
        at += pad16(floats * 4);
        return o;
    };
    if (w.segs > 1) {
        if (!p.segment_states) w.st = take(bh * w.segs * size);
        w.rt = take(bh * w.segs * size);
        w.decay = take(bh * w.segs);
    }
    if (p.nheads > p.n_groups) w.part = take(tok * p.dk);
    if (p.dlog_decay) {
        w.e = take(tok);
        w.a = take(tok);
        w.f = take(tok);
        w.ck = take(bh * w.blocks * size);
        w.y = take(bh * w.blocks * 4);
    }
    w.bytes = at;
    return w;
}

template <typename T>
static int run_bwd(const mm_linattn_bwd_params &p, hipStream_t s) {
    const BwdPlan w = plan_bwd(p);
    char *ws = static_cast<char *>(p.workspace);
    auto f32 = [&](int64_t o) { return reinterpret_cast<float *>(ws + o); };
    const int share = int(p.nheads / p.n_groups);
    const int64_t bh = p.batch * p.nheads, size = p.dk * p.dv;
    const View q = view(p.q, p.itype, p.q_batch_stride, p.q_seq_stride, p.q_group_stride, share, p.dk);
    const View k = view(p.k, p.itype, p.k_batch_stride, p.k_seq_stride, p.k_group_stride, share, p.dk);
    const View v = view(p.v, p.itype, p.v_batch_stride, p.v_seq_stride, p.v_head_stride, 1, p.dv);
    const View d = view(p.dout, p.itype, p.do_batch_stride, p.do_seq_stride, p.do_head_stride, 1, p.dv);
    const bool want_g = p.dlog_decay != nullptr, shared = share > 1;
    WalkArgs a = {};
    a.g = p.log_decay;
    a.gtype = p.gtype;
    a.g_batch = p.g_batch_stride; a.g_seq = p.g_seq_stride; a.g_head = p.g_head_stride;
    a.batch = p.batch; a.seqlen = p.seqlen; a.heads = p.nheads;
    a.segs = w.segs; a.seg_len = w.seg_len; a.blocks = w.blocks;
    if (w.segs > 1) {
        // The states the segments start from, and the states' gradients at their ends.
        a.seg_decay = f32(w.decay);
        a.kdim = int(p.dk); a.cdim = int(p.dv);
        if (!p.segment_states) {
            a.y = k; a.v = v; a.st = f32(w.st); a.scale = 1.f;
            if (const int rc = launch_segments<T>(a, false, s)) return rc;
            if (const int rc = launch_join(a.st, a.seg_decay, p.initial_state, a.segs, size, bh, false, s)) return rc;
        }
        a.y = q; a.v = d; a.st = f32(w.rt); a.scale = p.scale;
        if (const int rc = launch_segments<T>(a, true, s)) return rc;
        if (const int rc = launch_join(a.st, a.seg_decay, p.dlast_state, a.segs, size, bh, true, s)) return rc;
    }
    // dq: the forward walk with (do, v, k), its state the transposed one.
    a.x = d; a.y = v; a.v = k; a.z = q;
    a.kdim = int(p.dv); a.cdim = int(p.dk);
    a.scale = p.scale;
    const float *start = w.segs == 1 ? p.initial_state : p.segment_states ? static_cast<const float *>(p.segment_states) : f32(w.st);
    a.s0 = State{const_cast<float *>(start), 1, p.dv};
    a.s0_step = size;
    a.out = shared ? static_cast<void *>(f32(w.part)) : p.dq;
    a.out_f32 = shared;
    a.out_vec = view(p.dq, p.itype, 0, 0, 0, 1, p.dk).vec;
    a.out_batch = p.seqlen * p.nheads * p.dk; a.out_seq = p.nheads * p.dk; a.out_head = p.dk;
    if (want_g) {
        a.e = f32(w.e);
        a.ck = f32(w.ck);
        a.ck_last = p.dlast_state != nullptr;
    }
    if (const int rc = launch_walk<T>(a, want_g, s)) return rc;
    if (shared)
        if (const int rc = launch_head_sum(f32(w.part), p.dq, p.itype, p.batch * p.seqlen, int(p.nheads), share, int(p.dk), s)) return rc;
    BwdArgs r = {};
    r.q = q; r.k = k; r.v = v; r.dout = d;
    r.g = p.log_decay;
    r.gtype = p.gtype;
    r.g_batch = p.g_batch_stride; r.g_seq = p.g_seq_stride; r.g_head = p.g_head_stride;
    r.batch = p.batch; r.seqlen = p.seqlen; r.heads = p.nheads;
    r.dk = int(p.dk); r.dv = int(p.dv); r.segs = w.segs; r.seg_len = w.seg_len;
    r.scale = p.scale;
    r.r0 = w.segs > 1 ? f32(w.rt) : p.dlast_state;
    r.dr = p.dinitial_state;
    r.dv_out = p.dv_out;
    r.dk_out = shared ? static_cast<void *>(f32(w.part)) : p.dk_out;
    r.dk_f32 = shared;
    r.out_vec = view(p.dv_out, p.itype, 0, 0, 0, 1, p.dv).vec && view(p.dk_out, p.itype, 0, 0, 0, 1, p.dk).vec;
    r.blocks = w.blocks;
    r.has_last = p.dlast_state != nullptr;
    if (want_g) {
        r.a = f32(w.a);
        r.f = f32(w.f);
        r.ck = f32(w.ck);
        r.y = f32(w.y);
    }
    if (const int rc = launch_bwd<T>(r, s)) return rc;
    if (shared)
        if (const int rc = launch_head_sum(f32(w.part), p.dk_out, p.itype, p.batch * p.seqlen, int(p.nheads), share, int(p.dk), s)) return rc;
    if (want_g) return launch_decay_grad(r, f32(w.e), chunk_of(p.itype), p.decay_per_head != 0, p.dlog_decay, p.gtype, s);
    return MM_OK;
}

}  // namespace la
}  // namespace mm

using namespace mm;

extern "C" int64_t mm_linattn_fwd_workspace_size(const mm_linattn_fwd_params *p) {
    if (!p || p->batch <= 0 || p->seqlen <= 0 || p->nheads <= 0) return 0;
    int segs;
    int64_t len;
    la::segments(p->batch * p->nheads, p->seqlen, p->dk * p->dv, &segs, &len);
    return la::fwd_bytes(*p, segs);
}

extern "C" int64_t mm_linattn_bwd_workspace_size(const mm_linattn_bwd_params *p) {
    if (!p || p->batch <= 0 || p->seqlen <= 0 || p->nheads <= 0) return 0;
    return la::plan_bwd(*p).bytes;
}

extern "C" int mm_linattn_fwd(const mm_linattn_fwd_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_fwd: params is NULL");
    const mm_linattn_fwd_params &p = *params;
    if (const int rc = la::check(p.batch, p.seqlen, p.n_groups, p.nheads, p.dk, p.dv, p.itype, p.gtype, la::kMostPairs)) return rc;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int64_t bh = p.batch * p.nheads;
    if (bh == 0) return MM_OK;
    if (p.seqlen == 0) return p.last_state ? la::launch_copy(p.last_state, p.initial_state, bh * p.dk * p.dv, s) : MM_OK;
    if (!p.q || !p.k || !p.v || !p.log_decay || !p.out)
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_fwd: q, k, v, log_decay and out are required");
    if (!la::near({p.q_seq_stride, p.k_seq_stride, p.v_seq_stride, p.out_seq_stride}))
        return set_error(MM_ERR_UNSUPPORTED, "mm_linattn_fwd: sequence strides must be between 0 and 2^22 - 1 elements");
    switch (p.itype) {
        case MM_FLOAT32: return la::run_fwd<float>(p, s);
        case MM_FLOAT16: return la::run_fwd<f16_t>(p, s);
        default: return la::run_fwd<bf16_t>(p, s);
    }
}

extern "C" int mm_linattn_bwd(const mm_linattn_bwd_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_bwd: params is NULL");
    const mm_linattn_bwd_params &p = *params;
    if (const int rc = la::check(p.batch, p.seqlen, p.n_groups, p.nheads, p.dk, p.dv, p.itype, p.gtype, la::kMostPairs)) return rc;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int64_t bh = p.batch * p.nheads;
    if (bh == 0 || p.seqlen == 0) {
        if (bh > 0 && p.dinitial_state)
            if (const int rc = la::launch_copy(p.dinitial_state, p.dlast_state, bh * p.dk * p.dv, s)) return rc;
        if (p.dlog_decay && p.decay_per_head && p.nheads > 0) return la::launch_zero_g(p.dlog_decay, p.gtype, p.nheads, s);
        // Without heads nothing reaches q and k, which still have rows: empty sums.
        const int64_t n = p.nheads == 0 ? p.batch * p.seqlen * p.n_groups * p.dk : 0;
        if (n > 0) {
            if (!p.dq || !p.dk_out) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_bwd: dq and dk_out are required");
            if (const int rc = la::launch_zero_g(p.dq, p.itype, n, s)) return rc;
            return la::launch_zero_g(p.dk_out, p.itype, n, s);
        }
        return MM_OK;
    }
    if (!p.q || !p.k || !p.v || !p.log_decay || !p.dout || !p.dq || !p.dk_out || !p.dv_out)
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_bwd: q, k, v, log_decay, dout, dq, dk_out and dv_out are required");
    const int64_t need = la::plan_bwd(p).bytes;
    if (need > 0 && (!p.workspace || p.workspace_bytes < need))
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_bwd: the workspace is smaller than mm_linattn_bwd_workspace_size()");
    if (!la::near({p.q_seq_stride, p.k_seq_stride, p.v_seq_stride, p.do_seq_stride, p.nheads * p.dk, p.nheads * p.dv}))
        return set_error(MM_ERR_UNSUPPORTED, "mm_linattn_bwd: sequence strides must be between 0 and 2^22 - 1 elements");
    switch (p.itype) {
        case MM_FLOAT32: return la::run_bwd<float>(p, s);
        case MM_FLOAT16: return la::run_bwd<f16_t>(p, s);
        default: return la::run_bwd<bf16_t>(p, s);
    }
}

extern "C" int mm_linattn_update(const mm_linattn_update_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_update: params is NULL");
    const mm_linattn_update_params &p = *params;
    if (const int rc = la::check(p.batch, 1, p.n_groups, p.nheads, p.dk, p.dv, p.itype, p.gtype, la::kMostTokenPairs)) return rc;
    if (p.batch * p.nheads == 0) return MM_OK;
    if (!p.state || !p.q || !p.k || !p.v || !p.log_decay || !p.out)
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_update: state, q, k, v, log_decay and out are required");
    if (!la::apart(p)) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_linattn_update: elements of the state overlap");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (p.itype) {
        case MM_FLOAT32: return la::launch_update<float>(p, s);
        case MM_FLOAT16: return la::launch_update<f16_t>(p, s);
        default: return la::launch_update<bf16_t>(p, s);
    }
}
