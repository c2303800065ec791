// mm_delta_api.hip -- the gated delta rule's C entries: argument checks, the plan of a call (workspace), and the single-token kernel.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdlib>
#include <initializer_list>

#include "mm_common.h"
#include "mm_delta.h"
#include "mm_delta_host.h"
#include "mm_internal.h"

namespace mm {
namespace dr {

// ---- one token -----------------------------------------------------------------------------------

__device__ __forceinline__ float read_gate(const void *p, mm_dtype t, int64_t i) {
    switch (t) {
        case MM_FLOAT32: return reinterpret_cast<const float *>(p)[i];
        case MM_FLOAT16: return to_f32(reinterpret_cast<const f16_t *>(p)[i]);
        default: return to_f32(reinterpret_cast<const bf16_t *>(p)[i]);
    }
}

// Sums over the rows of a workgroup of each lane's four columns: over those that a wave holds, then over the waves, eight in pairs:
// what four of twice the rows add. So a pair's bits do not depend on how many pairs a call has (launch_update).
template <int LPR, int NW>
__device__ __forceinline__ void row_sums(float (&x)[4], float4 (*part)[LPR]) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int d = LPR; d < 64; d *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], d);
    if (tid % 64 < LPR) part[tid / 64][tid % LPR] = make_float4(x[0], x[1], x[2], x[3]);
    __syncthreads();
    x[0] = x[1] = x[2] = x[3] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w += NW / 4) {
        float4 y = part[w][tid % LPR];
        if constexpr (NW == 8) {
            const float4 y2 = part[w + 1][tid % LPR];
            y.x += y2.x; y.y += y2.y; y.z += y2.z; y.w += y2.w;
        }
        x[0] += y.x; x[1] += y.y; x[2] += y.z; x[3] += y.w;
    }
}

// S' = exp(g) S, u = beta (v - S'^T k), S = S' + k u^T, o = scale S^T q. Bound by the state, read once and written once: a workgroup
// holds one (batch row, head)'s columns of it (4 LPR of them) in registers between the two. LPR lanes cover a row in 16-byte pieces, RPT
// rows each. 256 x 40 heads of 128 x 128: 269 us, 1.34 GB at 5.0 TB/s (a large copy reaches 5.2); with twice the rows per lane and so half
// the workgroups on a CU 304, with waves of 32 columns that meet no other 359 (on a card where the first took 276).
template <typename T, int LPR, int RPT>
__global__ void __launch_bounds__(512) dr_update(const mm_delta_update_params p, int slices) {
    constexpr int NT = LPR == 32 ? 512 : 256, ROWS = NT / LPR;
    __shared__ float4 part[2][NT / 64][LPR];
    __shared__ float kq[2][MM_DELTA_MAX_DIM];
    const int64_t bh = blockIdx.x / unsigned(slices), b = bh / p.nheads, h = bh % p.nheads, grp = h / (p.nheads / p.n_groups);
    const int tid = threadIdx.x, x = 4 * (tid % LPR + LPR * int(blockIdx.x % unsigned(slices))), row0 = tid / LPR;
    const int dk = int(p.dk), dv = int(p.dv);
    float *s = p.state + b * p.state_batch_stride + h * p.state_head_stride + x;
    const T *q = reinterpret_cast<const T *>(p.q) + b * p.q_batch_stride + grp * p.q_group_stride;
    const T *k = reinterpret_cast<const T *>(p.k) + b * p.k_batch_stride + grp * p.k_group_stride;
    const T *v = reinterpret_cast<const T *>(p.v) + b * p.v_batch_stride + h * p.v_head_stride + x;
    const int n = dv - x < 4 ? dv - x : 4;    // elements of this lane's piece
    const bool vec = n == 4 && (reinterpret_cast<uintptr_t>(p.state) | p.state_dk_stride * 4 | p.state_head_stride * 4 | p.state_batch_stride * 4) % 16 == 0;
    // k and q first: their way through LDS does not wait for the state's rows then.
    const int at = tid % MM_DELTA_MAX_DIM;
    const float own = tid < 2 * MM_DELTA_MAX_DIM && at < dk ? to_f32((tid < MM_DELTA_MAX_DIM ? k : q)[at]) : 0.f;
    float w[RPT][4];
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
        const int row = row0 + r * ROWS;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[r][e] = 0.f;
        if (row < dk) {
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
    float u[4], o[4] = {0.f, 0.f, 0.f, 0.f}, z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = e < n ? to_f32(v[e]) : 0.f;
    float g = p.log_decay ? read_gate(p.log_decay, p.gtype, b * p.g_batch_stride + h * p.g_head_stride) : 0.f;
    g = p.log_decay ? expf(g < -128.f ? -128.f : g) : 1.f;
    const float beta = read_gate(p.beta, p.btype, b * p.b_batch_stride + h * p.b_head_stride);
    if (tid < 2 * MM_DELTA_MAX_DIM) kq[tid / MM_DELTA_MAX_DIM][at] = own;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
        const float kk = kq[0][row0 + r * ROWS], gr = row0 + r * ROWS < dk ? g : 0.f;   // rows past dk stay 0 whatever the growth
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[r][e] *= gr;
            z[e] = __builtin_fmaf(kk, w[r][e], z[e]);
        }
    }
    row_sums<LPR, NT / 64>(z, part[0]);
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = beta * (u[e] - z[e]);
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
        const int row = row0 + r * ROWS;
        if (row >= dk) continue;
        const float kk = kq[0][row], qq = kq[1][row];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[r][e] = __builtin_fmaf(kk, u[e], w[r][e]);
            o[e] = __builtin_fmaf(qq, w[r][e], o[e]);
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
    row_sums<LPR, NT / 64>(o, part[1]);
    if (tid < LPR && n > 0) {
        T *out = reinterpret_cast<T *>(p.out) + bh * dv + x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) out[e] = from_f32<T>(o[e] * p.scale);
    }
}

template <typename T>
static int launch_update(const mm_delta_update_params &p, hipStream_t s) {
    auto go = [&](auto lpr) {
        constexpr int LPR = decltype(lpr)::value, NT = LPR == 32 ? 512 : 256, RPT = 128 * LPR / NT;
        const int slices = int((p.dv + 4 * LPR - 1) / (4 * LPR));
        const dim3 grid(unsigned(p.batch * p.nheads * slices));
        if (p.dk <= 64) hipLaunchKernelGGL((dr_update<T, LPR, RPT / 2>), grid, dim3(NT), 0, s, p, slices);
        else hipLaunchKernelGGL((dr_update<T, LPR, RPT>), grid, dim3(NT), 0, s, p, slices);
        return launch_status("dr_update");
    };
    if (p.dv <= 32) return go(std::integral_constant<int, 8>{});
    // Whole rows, but halves of them where the pairs leave CUs without work (40 pairs of 128 x 128: 6.5 us, 7.4 whole).
    if (p.dv <= 64 || p.batch * p.nheads * 2 <= device_simds() / 4) return go(std::integral_constant<int, 16>{});
    return go(std::integral_constant<int, 32>{});
}

// dlog_decay[h] = sum over batch rows and tokens, one workgroup per head.
__global__ void __launch_bounds__(256) dr_decay_sum(const float *tmp, int64_t batch, int64_t heads, int64_t seqlen, void *out, mm_dtype gtype) {
    __shared__ float part[256];
    const int64_t h = blockIdx.x;
    float s = 0.f;
    for (int64_t b = 0; b < batch; ++b)
        for (int64_t t = threadIdx.x; t < seqlen; t += 256) s += tmp[(b * heads + h) * seqlen + t];
    part[threadIdx.x] = s;
    for (int n = 128; n > 0; n /= 2) {
        __syncthreads();
        if (int(threadIdx.x) < n) part[threadIdx.x] += part[threadIdx.x + n];
    }
    if (threadIdx.x) return;
    switch (gtype) {
        case MM_FLOAT32: reinterpret_cast<float *>(out)[h] = part[0]; break;
        case MM_FLOAT16: reinterpret_cast<f16_t *>(out)[h] = from_f32<f16_t>(part[0]); break;
        default: reinterpret_cast<bf16_t *>(out)[h] = from_f32<bf16_t>(part[0]);
    }
}

// ---- the plan of a call --------------------------------------------------------------------------

static int64_t size_of(mm_dtype t) { return t == MM_FLOAT32 ? 4 : 2; }
static bool known(mm_dtype t) { return t == MM_FLOAT32 || t == MM_FLOAT16 || t == MM_BFLOAT16; }
static int64_t pad16(int64_t n) { return (n + 15) / 16 * 16; }
static int64_t pad64(int64_t n) { return (n + 63) / 64 * 64; }

constexpr int64_t kMostPairs = int64_t(1) << 20, kMostTokenPairs = (int64_t(1) << 23) - 1;   // a launch takes less than 2^32 threads, one token's up to 512 for each

static View view(const void *p, mm_dtype t, int64_t b, int64_t s, int64_t h, int share, int64_t d) {
    const int64_t e = size_of(t);
    const bool vec = (reinterpret_cast<uintptr_t>(p) | b * e | s * e | h * e | d * e) % 16 == 0;
    return View{p, b, s, h, share, vec ? 1 : 0};
}

template <typename P>
static int check(const P &p, int64_t seqlen, int64_t pairs) {
    if (!known(p.itype) || !known(p.gtype) || !known(p.btype)) return set_error(MM_ERR_INVALID_ARGUMENT, "delta rule: unknown dtype");
    if (p.batch < 0 || seqlen < 0 || p.nheads < 0 || p.dk < 0 || p.dv < 0) return set_error(MM_ERR_INVALID_ARGUMENT, "delta rule: negative size");
    if (p.n_groups < 1 || p.nheads % p.n_groups) return set_error(MM_ERR_INVALID_ARGUMENT, "delta rule: nheads must be a multiple of n_groups");
    if (p.dk < 1 || p.dv < 1) return set_error(MM_ERR_INVALID_ARGUMENT, "delta rule: dk and dv must be at least 1");
    if (p.dk > MM_DELTA_MAX_DIM || p.dv > MM_DELTA_MAX_DIM) return set_error(MM_ERR_UNSUPPORTED, "delta rule: dk and dv must be <= 128");
    if (p.batch > pairs || p.nheads > pairs || p.batch * p.nheads > pairs)
        return set_error(MM_ERR_UNSUPPORTED, "delta rule: batch * nheads is too large (at most 2^20, for one token 2^23 - 1)");
    if (seqlen > (int64_t(1) << 23)) return set_error(MM_ERR_UNSUPPORTED, "delta rule: seqlen must be <= 2^23");
    return MM_OK;
}

// A size query has something to count: the plan's arithmetic is for calls that are not refused.
template <typename P>
static bool asks(const P *p) {
    return p && p->batch > 0 && p->seqlen > 0 && p->nheads > 0 && check(*p, p->seqlen, kMostPairs) == MM_OK;
}

// A tile's rows are addressed with 32-bit offsets.
static bool near(std::initializer_list<int64_t> strides) {
    for (const int64_t s : strides)
        if (s < 0 || s >= (int64_t(1) << 22)) return false;
    return true;
}

// No two elements of a state lie in one place: workgroups write them in any order. Each dimension has to step over all that the
// smaller ones span, as views of a contiguous tensor by slices and transposes do.
static bool apart(const mm_delta_update_params &p) {
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

// What forward and backward have alike.
template <typename P>
static Args common(const P &p) {
    Args a = {};
    const int share = int(p.nheads / p.n_groups), C = chunk_tokens(p.itype);
    a.q = view(p.q, p.itype, p.q_batch_stride, p.q_seq_stride, p.q_group_stride, share, p.dk);
    a.k = view(p.k, p.itype, p.k_batch_stride, p.k_seq_stride, p.k_group_stride, share, p.dk);
    a.v = view(p.v, p.itype, p.v_batch_stride, p.v_seq_stride, p.v_head_stride, 1, p.dv);
    a.g = Gate{p.log_decay, p.gtype, p.g_batch_stride, p.g_seq_stride, p.g_head_stride};
    a.beta = Gate{p.beta, p.btype, p.b_batch_stride, p.b_seq_stride, p.b_head_stride};
    a.batch = p.batch; a.seqlen = p.seqlen; a.heads = p.nheads;
    a.chunks = (p.seqlen + C - 1) / C;
    a.dk = int(p.dk); a.dv = int(p.dv);
    a.slices = int(pad64(p.dv) / 64);
    a.scale = p.scale;
    a.s0 = p.initial_state;
    return a;
}

// Segments of a row.
struct Cut {
    int segs;
    int64_t len;   // tokens
};
// By the time that the passes over a row of n segments take, in chunks of one workgroup of dr_walk alone on its CU (two on a CU take
// 1.85 of that for both): the first walk over all segments but the last (0.85 of a chunk; slices of V's columns and of the map's), the
// join, and the walk itself. A training step (`train`) runs the backward's walks on the same segments: states (0.9) and R (1.6), R once
// more before that (1.3), and another join. The times are bfloat16's, of 64 tokens a chunk; the other types' chunks have 32 and up to twice
// the products, and no ratios of their own were taken.
// 24 pairs of 64 x 64, 32,768 tokens, float32: 709 us in segments, the walk alone 3,845 in one piece; 48 pairs, 1,777 tokens, bfloat16: 76,
// the walk alone 121. 160 pairs of 4,096 tokens go in one piece, 546 us, and so do the 192 of a training step.
static Cut segments(int64_t pairs, int64_t seqlen, int64_t dk, int64_t dv, mm_dtype t, bool train) {
    const int C = chunk_tokens(t);
    const int64_t chunks = (seqlen + C - 1) / C, cus = device_simds() / 4, vs = pad64(dv) / 64, ks = pad64(dk) / 64;
    auto cut = [&](int64_t n) {
        const int64_t per = (chunks + n - 1) / n;
        return Cut{int((chunks + per - 1) / per), per * C};
    };
    if (const char *e = std::getenv("MM_DELTA_SEGMENTS")) return cut(std::min<int64_t>({std::max<int64_t>(std::atoll(e), 1), chunks, kMostPairs / pairs}));
    const double us = (ks == 2 ? 4.8 : 3.6), join = (ks == 2 ? 3.0 : 1.2) / us, launch = 6.0 / us;
    auto rounds = [&](int64_t groups) {
        const int64_t full = groups / (2 * cus), rest = groups % (2 * cus);
        return 1.85 * double(full) + (rest == 0 ? 0.0 : rest <= cus ? 1.0 : 1.85);
    };
    Cut best = cut(1);
    double least = 0.0;
    for (int64_t n = 1; n <= std::min<int64_t>({chunks / 2 + 1, 64, kMostPairs / pairs}); ++n) {
        const Cut c = cut(n);
        if (c.segs != n) continue;
        const double m = double(c.len / C), walk = rounds(pairs * n * vs);
        double cost = m * walk * (train ? 1.0 + 0.9 + 1.6 : 1.0);
        if (n > 1) {
            cost += m * 0.85 * rounds(pairs * (n - 1) * vs + pairs * (train ? n : n - 1) * ks) + double(n) * join + 2.0 * launch;
            if (train) cost += m * 1.3 * rounds(pairs * (n - 1) * vs) + double(n) * join + 2.0 * launch;
        }
        if (n == 1 || cost < least) {
            least = cost;
            best = c;
        }
    }
    return best;
}

// Bytes taken from a workspace, one piece after the other.
struct Take {
    int64_t at = 0;
    int64_t operator()(int64_t bytes) {
        const int64_t o = at;
        at += pad16(bytes);
        return o;
    }
};

// What a training step's forward leaves of its segments for the backward: maps, starts.
struct Kept {
    Cut cut;
    int64_t maps, starts, flags, bytes;   // byte offsets
};
template <typename P>
static Kept plan_kept(const P &p, bool train) {
    Kept w = {};
    const int64_t bh = p.batch * p.nheads, kd = pad64(p.dk), vd = pad64(p.dv);
    w.cut = segments(bh, p.seqlen, p.dk, p.dv, p.itype, train);
    if (w.cut.segs == 1) return w;
    Take take;
    w.maps = take(bh * w.cut.segs * kd * (vd + kd) * 4);
    w.starts = take(bh * w.cut.segs * kd * vd * 4);
    w.flags = take(bh * 4);
    w.bytes = take.at;
    return w;
}
template <typename P>
static int check_kept(const P &p) {
    if (!p.segment_states || p.segment_states_bytes == plan_kept(p, true).bytes) return MM_OK;
    return set_error(MM_ERR_INVALID_ARGUMENT, "delta rule: segment_states is not of mm_delta_segment_states_size()");
}
static void set_kept(Args &a, const Kept &w, void *place) {
    char *at = static_cast<char *>(place);
    a.segs = w.cut.segs;
    a.seg_len = w.cut.len;
    a.maps = reinterpret_cast<float *>(at + w.maps);
    a.starts = reinterpret_cast<float *>(at + w.starts);
    a.flags = reinterpret_cast<int *>(at + w.flags);
}

static int64_t records(const mm_delta_fwd_params &p) {
    const int C = chunk_tokens(p.itype);
    return p.batch * p.nheads * ((p.seqlen + C - 1) / C) * record_bytes(C, 2);
}
static int64_t fwd_bytes(const mm_delta_fwd_params &p) { return records(p) + (p.segment_states ? 0 : plan_kept(p, false).bytes); }

template <typename T>
static int run_fwd(const mm_delta_fwd_params &p, hipStream_t s) {
    Args a = common(p);
    a.rec_a = static_cast<char *>(p.workspace);
    a.rec_a_step = int(record_bytes(chunk_tokens(p.itype), 2));
    if (p.segment_states) set_kept(a, plan_kept(p, true), p.segment_states);
    else set_kept(a, plan_kept(p, false), static_cast<char *>(p.workspace) + records(p));
    a.last_map = p.segment_states != nullptr;
    a.s1 = p.last_state;
    a.out = p.out;
    a.out_vec = view(p.out, p.itype, p.out_batch_stride, p.out_seq_stride, p.out_head_stride, 1, p.dv).vec;
    a.out_batch = p.out_batch_stride; a.out_seq = p.out_seq_stride; a.out_head = p.out_head_stride;
    if (const int rc = launch_prep<T>(a, false, s)) return rc;
    return launch_walk<T>(a, false, s);
}

// The backward's workspace, in order.
struct BwdPlan {
    Kept kept;
    int64_t rec_a, rec_b, states, z, r, dx, pbeta, dq, dk, dg, segs, back_maps, back_starts, bytes;   // byte offsets
};

static BwdPlan plan_bwd(const mm_delta_bwd_params &p) {
    BwdPlan w = {};
    const int C = chunk_tokens(p.itype);
    const int64_t bh = p.batch * p.nheads, chunks = (p.seqlen + C - 1) / C, kd = pad64(p.dk), vd = pad64(p.dv);
    w.kept = plan_kept(p, true);
    Take take;
    w.rec_a = take(bh * chunks * record_bytes(C, 1));
    w.rec_b = take(bh * chunks * record_bytes(C, 2));
    w.states = take(bh * chunks * kd * vd * 4);
    w.z = take(bh * chunks * C * vd * 4);
    w.r = take(bh * chunks * kd * vd * 4);
    w.dx = take(bh * chunks * C * vd * 4);
    w.pbeta = take(vd / 64 * bh * chunks * C * 4);
    if (p.nheads > p.n_groups) {
        w.dq = take(bh * p.seqlen * p.dk * 4);
        w.dk = take(bh * p.seqlen * p.dk * 4);
    }
    if (p.dlog_decay && p.decay_per_head) w.dg = take(bh * p.seqlen * 4);
    if (w.kept.cut.segs > 1) {
        w.back_maps = take(bh * w.kept.cut.segs * kd * vd * 4);
        w.back_starts = take(bh * w.kept.cut.segs * kd * vd * 4);
        if (!p.segment_states) w.segs = take(w.kept.bytes);
    }
    w.bytes = take.at;
    return w;
}

template <typename T>
static int run_bwd(const mm_delta_bwd_params &p, hipStream_t s) {
    const BwdPlan w = plan_bwd(p);
    char *ws = static_cast<char *>(p.workspace);
    auto f32 = [&](int64_t o) { return reinterpret_cast<float *>(ws + o); };
    const int share = int(p.nheads / p.n_groups);
    const bool shared = share > 1;
    Args a = common(p);
    a.dout = view(p.dout, p.itype, p.do_batch_stride, p.do_seq_stride, p.do_head_stride, 1, p.dv);
    a.rec_a = ws + w.rec_a;
    a.rec_a_step = int(record_bytes(chunk_tokens(p.itype), 1));
    a.rec_b = ws + w.rec_b;
    set_kept(a, w.kept, p.segment_states ? const_cast<void *>(p.segment_states) : ws + w.segs);
    a.kept_starts = p.segment_states != nullptr;
    a.last_map = 1;
    a.back_maps = f32(w.back_maps); a.back_starts = f32(w.back_starts);
    a.states = f32(w.states); a.z = f32(w.z); a.r = f32(w.r); a.dx = f32(w.dx); a.pbeta = f32(w.pbeta);
    a.dlast = p.dlast_state;
    a.ds0 = p.dinitial_state;
    a.out = p.dv_out;
    a.out_batch = p.seqlen * p.nheads * p.dv; a.out_seq = p.nheads * p.dv; a.out_head = p.dv;
    a.out_vec = view(p.dv_out, p.itype, 0, 0, 0, 1, p.dv).vec;
    a.dq = shared ? static_cast<void *>(f32(w.dq)) : p.dq;
    a.dk_out = shared ? static_cast<void *>(f32(w.dk)) : p.dk_out;
    a.dqk_f32 = shared;
    a.dqk_vec = view(p.dq, p.itype, 0, 0, 0, 1, p.dk).vec && view(p.dk_out, p.itype, 0, 0, 0, 1, p.dk).vec;
    a.dbeta = p.dbeta;
    if (p.dlog_decay) {
        if (p.decay_per_head) a.dg_sum = f32(w.dg);
        else a.dg = p.dlog_decay;
    }
    if (const int rc = launch_prep<T>(a, true, s)) return rc;
    if (const int rc = launch_walk<T>(a, true, s)) return rc;
    if (const int rc = launch_back<T>(a, s)) return rc;
    if (const int rc = launch_grad<T>(a, s)) return rc;
    if (shared) {
        if (const int rc = la::launch_head_sum(f32(w.dq), p.dq, p.itype, p.batch * p.seqlen, int(p.nheads), share, int(p.dk), s)) return rc;
        if (const int rc = la::launch_head_sum(f32(w.dk), p.dk_out, p.itype, p.batch * p.seqlen, int(p.nheads), share, int(p.dk), s)) return rc;
    }
    if (!a.dg_sum) return MM_OK;
    hipLaunchKernelGGL(dr_decay_sum, dim3(unsigned(p.nheads)), dim3(256), 0, s, a.dg_sum, p.batch, p.nheads, p.seqlen, p.dlog_decay, p.gtype);
    return launch_status("dr_decay_sum");
}

}  // namespace dr
}  // namespace mm

using namespace mm;

extern "C" int64_t mm_delta_fwd_workspace_size(const mm_delta_fwd_params *p) {
    if (!dr::asks(p)) return 0;
    return dr::fwd_bytes(*p);
}

extern "C" int64_t mm_delta_segment_states_size(const mm_delta_fwd_params *p) {
    if (!dr::asks(p)) return 0;
    return dr::plan_kept(*p, true).bytes;
}

extern "C" int64_t mm_delta_bwd_workspace_size(const mm_delta_bwd_params *p) {
    if (!dr::asks(p)) return 0;
    return dr::plan_bwd(*p).bytes;
}

extern "C" int mm_delta_fwd(const mm_delta_fwd_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_fwd: params is NULL");
    const mm_delta_fwd_params &p = *params;
    if (const int rc = dr::check(p, p.seqlen, dr::kMostPairs)) return rc;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int64_t bh = p.batch * p.nheads;
    if (bh == 0) return MM_OK;
    if (p.seqlen == 0) return p.last_state ? la::launch_copy(p.last_state, p.initial_state, bh * p.dk * p.dv, s) : MM_OK;
    if (!p.q || !p.k || !p.v || !p.beta || !p.out)
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_fwd: q, k, v, beta and out are required");
    if (const int rc = dr::check_kept(p)) return rc;
    if (!p.workspace || p.workspace_bytes < dr::fwd_bytes(p))
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_fwd: the workspace is smaller than mm_delta_fwd_workspace_size()");
    if (!dr::near({p.q_seq_stride, p.k_seq_stride, p.v_seq_stride, p.out_seq_stride}))
        return set_error(MM_ERR_UNSUPPORTED, "mm_delta_fwd: sequence strides must be between 0 and 2^22 - 1 elements");
    switch (p.itype) {
        case MM_FLOAT32: return dr::run_fwd<float>(p, s);
        case MM_FLOAT16: return dr::run_fwd<f16_t>(p, s);
        default: return dr::run_fwd<bf16_t>(p, s);
    }
}

extern "C" int mm_delta_bwd(const mm_delta_bwd_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_bwd: params is NULL");
    const mm_delta_bwd_params &p = *params;
    if (const int rc = dr::check(p, p.seqlen, dr::kMostPairs)) return rc;
    if (p.dlog_decay && !p.log_decay) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_bwd: dlog_decay goes with log_decay");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int64_t bh = p.batch * p.nheads;
    if (bh == 0 || p.seqlen == 0) {
        if (bh > 0 && p.dinitial_state)
            if (const int rc = la::launch_copy(p.dinitial_state, p.dlast_state, bh * p.dk * p.dv, s)) return rc;
        if (p.dlog_decay && p.decay_per_head && p.nheads > 0)
            if (const int rc = la::launch_zero_g(p.dlog_decay, p.gtype, p.nheads, s)) return rc;
        // Without heads nothing reaches q and k, which still have rows: empty sums.
        const int64_t n = p.nheads == 0 ? p.batch * p.seqlen * p.n_groups * p.dk : 0;
        if (n > 0) {
            if (!p.dq || !p.dk_out) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_bwd: dq and dk_out are required");
            if (const int rc = la::launch_zero_g(p.dq, p.itype, n, s)) return rc;
            return la::launch_zero_g(p.dk_out, p.itype, n, s);
        }
        return MM_OK;
    }
    if (!p.q || !p.k || !p.v || !p.beta || !p.dout || !p.dq || !p.dk_out || !p.dv_out || !p.dbeta)
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_bwd: q, k, v, beta, dout, dq, dk_out, dv_out and dbeta are required");
    if (const int rc = dr::check_kept(p)) return rc;
    if (!p.workspace || p.workspace_bytes < dr::plan_bwd(p).bytes)
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_bwd: the workspace is smaller than mm_delta_bwd_workspace_size()");
    if (!dr::near({p.q_seq_stride, p.k_seq_stride, p.v_seq_stride, p.do_seq_stride, p.nheads * p.dk, p.nheads * p.dv}))
        return set_error(MM_ERR_UNSUPPORTED, "mm_delta_bwd: sequence strides must be between 0 and 2^22 - 1 elements");
    switch (p.itype) {
        case MM_FLOAT32: return dr::run_bwd<float>(p, s);
        case MM_FLOAT16: return dr::run_bwd<f16_t>(p, s);
        default: return dr::run_bwd<bf16_t>(p, s);
    }
}

extern "C" int mm_delta_update(const mm_delta_update_params *params, void *stream) {
    if (!params) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_update: params is NULL");
    const mm_delta_update_params &p = *params;
    if (const int rc = dr::check(p, 1, dr::kMostTokenPairs)) return rc;
    if (p.batch * p.nheads == 0) return MM_OK;
    if (!p.state || !p.q || !p.k || !p.v || !p.beta || !p.out)
        return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_update: state, q, k, v, beta and out are required");
    if (!dr::apart(p)) return set_error(MM_ERR_INVALID_ARGUMENT, "mm_delta_update: elements of the state overlap");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (p.itype) {
        case MM_FLOAT32: return dr::launch_update<float>(p, s);
        case MM_FLOAT16: return dr::launch_update<f16_t>(p, s);
        default: return dr::launch_update<bf16_t>(p, s);
    }
}
